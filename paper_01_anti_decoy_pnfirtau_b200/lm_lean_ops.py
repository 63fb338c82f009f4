"""Operators of a decoder's training step that keep little for the backward pass,
on this library's tcgen05 kernels (csrc/gated.cu, csrc/xent_stream.cu, csrc/act8.cu
over the GEMM core csrc/gemm_tc.cuh). They stand beside ``mlp_gelu``,
``head_cross_entropy`` and ``Linear`` (lm_ops) of the Pre-LN decoder of the
reference's language-model experiments (experiments/exp4_wikitext2_lm.py:183-259).

- ``gated_linear``: ``act(x Wg^T + bg) * (x Wu^T + bu)`` (SwiGLU / GEGLU), both
  projections, the activation and the product in one kernel. The backward keeps x and
  the two pre-activations, or with ``checkpoint_8bit`` only x in 8 bits, from which it
  computes the pre-activations again. Calls of a few rows (single tokens) that need no
  gradient take the same entry.
- ``gated_mlp``: the block ``down(gated_linear(x))`` of three ``nn.Linear`` layers.
- ``streamed_cross_entropy``: the head's softmax cross entropy without its logits: the
  forward keeps one number per row, the backward computes the logits again for one
  piece of the vocabulary at a time.
- ``act8_pack`` / ``act8_unpack`` / ``act8_weight_grad``: an activation in 8 bits (e4m3
  with a power of two per row and 128 columns) and the weight gradient that reads it;
  ``lm_ops.Linear`` uses them when its ``checkpoint_8bit`` is set.

Operands are bfloat16 or float16: under CUDA autocast the inputs are cast to the
autocast dtype, else the input's dtype counts; float32 without autocast raises. CUDA
only; a CPU tensor raises. Results are bitwise reproducible on a given GPU.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn

from . import _lib
from .pnfirtau_ops import _DTYPES, _check_pending, _ptr, _require_cuda, _status_ptr, _stream

_ACTS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
_TYPES16 = (torch.bfloat16, torch.float16)


def _compute_dtype(x: torch.Tensor, what: str) -> torch.dtype:
    dt = torch.get_autocast_dtype("cuda") if x.is_cuda and torch.is_autocast_enabled("cuda") else x.dtype
    if dt not in _TYPES16:
        raise RuntimeError(f"{what}: bfloat16 or float16 expected (or CUDA autocast to one of them), got {dt}")
    return dt


def _workspace(nbytes: int, dev: torch.device) -> torch.Tensor:
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)


def _pad8(n: int) -> int:
    return (n + 7) // 8 * 8


def _rows16(t: torch.Tensor, dt: torch.dtype) -> torch.Tensor:
    """``t`` (2-D) in ``dt`` as rows that a TMA map takes: unit column stride, row stride
    a multiple of 8 elements, 16-byte base. A view of ``t`` when it is that already."""
    if t.dtype != dt:
        t = t.to(dt)
    rows, cols = t.shape
    ld = _ld(t)
    if (t.stride(1) == 1 or cols == 1) and t.data_ptr() % 16 == 0 and ld % 8 == 0 and ld >= cols:
        return t
    if t.stride(1) != 1 and cols > 1:
        t = t.contiguous()
    out = torch.empty((rows, _pad8(cols)), dtype=dt, device=t.device)[:, :cols]
    _lib.check(_lib.lib().pnft_copy_rows16(t.data_ptr(), t.stride(0), out.data_ptr(), _pad8(cols), rows, cols,
                                           _stream(t.device)), "pnft_copy_rows16")
    return out


def _ld(t: torch.Tensor) -> int:
    """Row stride of a matrix; a single row's is free, so its padded width."""
    return t.stride(0) if t.shape[0] > 1 else _pad8(t.shape[1])


# ---------------------------------------------------------------- 8-bit activations
@dataclass(frozen=True)
class Act8:
    """An activation in 8 bits: ``q`` (e4m3 bytes, ``[M, D]`` padded to a multiple of 16
    columns), ``exponents`` (int8, one per row and 128 columns), and the packed tensor's
    shape and dtype. The value of an element is ``q * 2^exponent``."""

    q: torch.Tensor
    exponents: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    @property
    def width(self) -> int:
        return self.shape[-1]

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.exponents.numel()


def act8_pack(x: torch.Tensor) -> Act8:
    """``x`` (float32, bfloat16 or float16; ``[..., D]``) in 8 bits: per row and block of
    128 columns e4m3 values times the least power of two that brings the block's largest
    magnitude to 448 or less, rounded to nearest even. NaN and infinities become NaN."""
    dev = _require_cuda("act8_pack", x)
    if x.dtype not in _DTYPES:
        raise RuntimeError(f"act8_pack: float32, bfloat16 or float16 expected, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError(f"act8_pack: rows of at least one column expected, got {tuple(x.shape)}")
    D = x.shape[-1]
    x2 = x.detach().reshape(-1, D)
    if x2.stride(1) != 1 or x2.stride(0) < D:
        x2 = x2.contiguous()
    M, nb = x2.shape[0], (D + 127) // 128
    q = torch.empty((M, (D + 15) // 16 * 16), dtype=torch.uint8, device=dev)
    e = torch.empty((M, nb), dtype=torch.int8, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().pnft_act8_pack(x2.data_ptr(), max(x2.stride(0), D), q.data_ptr(), q.shape[1], e.data_ptr(), nb, M, D,
                                             _DTYPES[x.dtype], _stream(dev)), "pnft_act8_pack")
    return Act8(q, e, x.shape, x.dtype)


def _act8_rows(p: Act8, dt: torch.dtype) -> torch.Tensor:
    """The values as rows ``[M, D]`` of ``dt`` whose stride is a multiple of 8."""
    M, D, dev = p.q.shape[0], p.width, p.q.device
    y = torch.empty((M, _pad8(D)), dtype=dt, device=dev)[:, :D]
    _lib.check(_lib.lib().pnft_act8_unpack(p.q.data_ptr(), p.q.shape[1], p.exponents.data_ptr(), p.exponents.shape[1],
                                           y.data_ptr(), _pad8(D), M, D, _DTYPES[dt], _stream(dev)), "pnft_act8_unpack")
    return y


def act8_unpack(p: Act8) -> torch.Tensor:
    """The tensor that ``p`` stands for, in the shape and dtype that were packed (exact:
    the dtype holds every packed value)."""
    with torch.cuda.device(p.q.device):
        return _act8_rows(p, p.dtype).reshape(p.shape)


def act8_weight_grad(dy: torch.Tensor, p: Act8, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``dy^T x`` for the packed ``x``: the weight gradient ``[N, D]`` of a Linear layer
    from its output's gradient ``dy`` (``[..., N]``, bfloat16 or float16, as many rows as
    ``x``) and its input kept in 8 bits; fp32 sums."""
    dev = _require_cuda("act8_weight_grad", dy, p.q)
    if dy.dtype not in _TYPES16:
        raise RuntimeError(f"act8_weight_grad: bfloat16 or float16 gradient expected, got {dy.dtype}")
    if dy.dtype == torch.float16 and p.dtype != torch.float16:
        raise RuntimeError(f"act8_weight_grad: a float16 gradient needs a float16 activation, got {p.dtype}")
    if dy.dim() == 0 or dy.shape[-1] == 0:
        raise RuntimeError(f"act8_weight_grad: rows of at least one column expected, got {tuple(dy.shape)}")
    dy2 = dy.detach().reshape(-1, dy.shape[-1])
    if dy2.shape[0] != p.q.shape[0]:
        raise RuntimeError(f"act8_weight_grad: {dy2.shape[0]} rows of gradient but {p.q.shape[0]} of activation")
    with torch.cuda.device(dev):
        return _weight_grads(_rows16(dy2, dy.dtype), _act8_rows(p, dy.dtype), (out_dtype,))[0]


def _weight_grads(dy: torch.Tensor, x: torch.Tensor, dtypes, split: int | None = None, rows: int | None = None):
    """``dy^T x`` (both from ``_rows16``) as one matrix, or as two of ``rows`` rows each
    that start at rows 0 and ``split`` of the product."""
    K, M = dy.shape
    N, dev = x.shape[1], dy.device
    two = split is not None
    split, rows = split or M, rows or M
    dt = dtypes[0]
    code = _DTYPES[dt]
    outs = [torch.empty((rows, N), dtype=dt, device=dev) for _ in range(2 if two else 1)]
    L = _lib.lib()
    nbytes = L.pnft_weight_grad_workspace_size(K, M, N)
    ws = _workspace(nbytes, dev)
    _lib.check(L.pnft_weight_grad(dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), outs[0].data_ptr(),
                                  outs[1].data_ptr() if two else None, N, split, rows, code, ws.data_ptr(), nbytes, K, M,
                                  N, _DTYPES[dy.dtype], _status_ptr(dev), _stream(dev)), "pnft_weight_grad")
    return outs


# ---------------------------------------------------------------- gated product
class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act: int, dt: torch.dtype, keep: str | None, pre=None):
        dev = x.device
        _check_pending(dev)
        D, F_ = wg.shape[1], wg.shape[0]
        with torch.cuda.device(dev):
            x2 = _rows16(x.reshape(-1, D), dt)
            wgc, wuc = (_rows16(w, dt) for w in (pre if pre is not None else (wg, wu)))
            M, L, st = x2.shape[0], _lib.lib(), _stream(dev)
            biases = _biases(bg, bu)
            h = torch.empty((M, F_), dtype=dt, device=dev)
            g = u = None
            if keep == "pre":
                Fp = _pad8(F_)
                g, u = torch.empty((2, M, Fp), dtype=dt, device=dev)
            _lib.check(L.pnft_gated_fwd(x2.data_ptr(), _ld(x2), wgc.data_ptr(), _ld(wgc), wuc.data_ptr(), _ld(wuc),
                                        *biases, h.data_ptr(), F_, _ptr(g), _ptr(u), 0 if g is None else g.stride(0), M, D,
                                        F_, act, _DTYPES[dt], _status_ptr(dev), st), "pnft_gated_fwd")
        if keep is not None:
            ctx.act8 = None
            if keep == "act8":
                p = act8_pack(x2)
                ctx.act8 = (p.shape, p.dtype)
                ctx.save_for_backward(p.q, p.exponents, None, None, wgc, wuc, bg, bu)
            else:
                ctx.save_for_backward(x2, None, g, u, wgc, wuc, bg, bu)
            ctx.act, ctx.dt, ctx.x_shape, ctx.x_dtype = act, dt, x.shape, x.dtype
            ctx.w_dtypes = (wg.dtype, wu.dtype)
        return h.view(*x.shape[:-1], F_)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        a, b, g, u, wg, wu, bg, bu = ctx.saved_tensors
        dt, dev = ctx.dt, wg.device
        F_, D = wg.shape
        L = _lib.lib()
        with torch.cuda.device(dev):
            st = _stream(dev)
            dh2 = _rows16(dh.reshape(-1, F_), dt)
            M = dh2.shape[0]
            Fp = _pad8(F_)
            x2 = a if ctx.act8 is None else _act8_rows(Act8(a, b, *ctx.act8), dt)
            need = ctx.needs_input_grad
            d = torch.empty((M, 2 * Fp), dtype=dt, device=dev)  # dg, du side by side: one weight-gradient product
            dg, du = d[:, :F_], d[:, Fp:Fp + F_]
            dbg = torch.empty(F_, dtype=bg.dtype, device=dev) if bg is not None and need[3] else None
            dbu = torch.empty(F_, dtype=bu.dtype, device=dev) if bu is not None and need[4] else None
            code, b_code = _DTYPES[dt], _b_code(bg, bu)
            sums = dbg is not None or dbu is not None
            nbytes = L.pnft_gated_bias_workspace_size(M, F_) if sums else 0
            ws = _workspace(nbytes, dev) if sums else None
            if ctx.act8 is None:
                _lib.check(L.pnft_gated_bwd_point(dh2.data_ptr(), _ld(dh2), g.data_ptr(), u.data_ptr(), g.stride(0),
                                                  dg.data_ptr(), du.data_ptr(), 2 * Fp, _ptr(dbg), _ptr(dbu), b_code, _ptr(ws),
                                                  nbytes, M, F_, ctx.act, code, st), "pnft_gated_bwd_point")
            else:
                _lib.check(L.pnft_gated_bwd_recompute(x2.data_ptr(), _ld(x2), wg.data_ptr(), _ld(wg), wu.data_ptr(), _ld(wu),
                                                      *_biases(bg, bu), dh2.data_ptr(), _ld(dh2), dg.data_ptr(),
                                                      du.data_ptr(), 2 * Fp, M, D, F_, ctx.act, code, _status_ptr(dev), st),
                           "pnft_gated_bwd_recompute")
                if sums:
                    _lib.check(L.pnft_gated_bwd_point(None, 0, dg.data_ptr(), du.data_ptr(), 2 * Fp, None, None, 0, _ptr(dbg),
                                                      _ptr(dbu), b_code, _ptr(ws), nbytes, M, F_, ctx.act, code, st),
                               "pnft_gated_bwd_point")
            dx = None
            if need[0]:
                dx = torch.empty((M, D), dtype=ctx.x_dtype, device=dev)
                nb = L.pnft_gated_dx_workspace_size(M, D, F_)
                ws2 = _workspace(nb, dev)
                _lib.check(L.pnft_gated_dx(dg.data_ptr(), du.data_ptr(), 2 * Fp, wg.data_ptr(), _ld(wg), wu.data_ptr(), _ld(wu),
                                           dx.data_ptr(), D, _DTYPES[ctx.x_dtype], ws2.data_ptr(), nb, M, D, F_, code,
                                           _status_ptr(dev), st), "pnft_gated_dx")
                dx = dx.view(ctx.x_shape)
            dwg = dwu = None
            if need[1] or need[2]:
                dwg, dwu = _weight_grads(d, x2, ctx.w_dtypes, split=Fp, rows=F_)
                dwg, dwu = (t if n else None for t, n in ((dwg, need[1]), (dwu, need[2])))
        return dx, dwg, dwu, dbg, dbu, None, None, None, None


def _b_code(bg, bu) -> int:
    b = bg if bg is not None else bu
    return _lib.DTYPE_F32 if b is None else _DTYPES[b.dtype]


def _biases(bg, bu):
    return _ptr(bg), _ptr(bu), _b_code(bg, bu)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, activation: str = "silu", *, checkpoint_8bit: bool = False,
                 casts=None) -> torch.Tensor:
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)``: ``x`` ``[..., D]``, the weights
    ``[F, D]`` (``nn.Linear``'s layout), ``activation`` ``"silu"`` or ``"gelu"`` (erf form).
    The result and the sums' operands have the autocast dtype under CUDA autocast, else
    ``x.dtype`` (bfloat16 or float16). Gradients of everything but ``activation``; twice
    differentiating raises.

    ``checkpoint_8bit``: the backward keeps ``x`` in 8 bits (``act8_pack``) and nothing else,
    and is the gradient at that 8-bit ``x``: it computes the pre-activations again from it.
    The forward's result does not change. ``casts``: an ``lm_ops.Bf16Casts`` with current
    bf16 copies of the weights, used when the dtype is bf16."""
    ts = [t for t in (x, w_gate, w_up, b_gate, b_up) if t is not None]
    _require_cuda("gated_linear", *ts)
    if activation not in _ACTS:
        raise ValueError(f"gated_linear: activation {activation!r} (one of {sorted(_ACTS)})")
    if x.dim() == 0 or w_gate.dim() != 2 or w_gate.shape != w_up.shape or x.shape[-1] != w_gate.shape[1]:
        raise RuntimeError(f"gated_linear: x {tuple(x.shape)}, weights {tuple(w_gate.shape)} and {tuple(w_up.shape)}: [..., D] "
                           "and twice [F, D] expected")
    if 0 in w_gate.shape:
        raise RuntimeError(f"gated_linear: empty weights {tuple(w_gate.shape)}")
    for b in (b_gate, b_up):
        if b is not None and b.shape != w_gate.shape[:1]:
            raise RuntimeError(f"gated_linear: bias {tuple(b.shape)} for {w_gate.shape[0]} columns")
    for t in ts:
        if t.dtype not in _DTYPES:
            raise RuntimeError(f"gated_linear: float32, bfloat16 or float16 tensors expected, got {t.dtype}")
    if w_gate.dtype != w_up.dtype or (b_gate is not None and b_up is not None and b_gate.dtype != b_up.dtype):
        raise RuntimeError("gated_linear: the two projections' parameters must have the same dtype")
    dt = _compute_dtype(x, "gated_linear")
    b_gate, b_up = (None if b is None else b.contiguous() for b in (b_gate, b_up))
    keep = None
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        keep = "act8" if checkpoint_8bit else "pre"
    pre = casts.lookup(w_gate, w_up) if casts is not None and dt == torch.bfloat16 else None
    return _GatedLinearFn.apply(x, w_gate, w_up, b_gate, b_up, _ACTS[activation], dt, keep, pre)


# ---------------------------------------------------------------- streamed cross entropy
class _StreamXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, targets, ignore_index: int, reduction: str, dt: torch.dtype, need: bool, pre=None):
        dev = h.device
        _check_pending(dev)
        V, D = weight.shape
        L = _lib.lib()
        with torch.cuda.device(dev):
            st = _stream(dev)
            h2 = h.reshape(-1, D)
            h2 = h2 if h2.dtype == dt else h2.to(dt)
            h2 = h2 if D == 1 or h2.stride(1) == 1 else h2.contiguous()
            w = _rows16(weight if pre is None else pre, dt)
            t = targets.reshape(-1).to(torch.int64).contiguous()
            M = h2.shape[0]
            Mp, Dp = (M + 127) // 128 * 128, _pad8(D)
            hc = torch.empty((Mp, Dp), dtype=dt, device=dev)
            saved = _workspace(L.pnft_stream_xent_saved_size(M), dev)
            rows = torch.empty(M, dtype=torch.float32, device=dev) if reduction == "none" else None
            loss = None if reduction == "none" else torch.empty((), dtype=torch.float32, device=dev)
            nbytes = L.pnft_stream_xent_fwd_workspace_size(M, V)
            ws = _workspace(nbytes, dev)
            _lib.check(L.pnft_stream_xent_fwd(h2.data_ptr(), max(h2.stride(0), D), w.data_ptr(), _ld(w), t.data_ptr(),
                                              ignore_index, hc.data_ptr(), Dp, saved.data_ptr(), _ptr(rows), _ptr(loss),
                                              reduction == "mean", ws.data_ptr(), nbytes, M, V, D, _DTYPES[dt],
                                              _status_ptr(dev), st), "pnft_stream_xent_fwd")
        if need:
            ctx.save_for_backward(hc, saved, w)
            ctx.M, ctx.dt, ctx.reduction, ctx.h_shape, ctx.h_dtype, ctx.w_dtype = M, dt, reduction, h.shape, h.dtype, weight.dtype
        return loss if rows is None else rows.view(targets.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        hc, saved, w = ctx.saved_tensors
        V, D = w.shape
        M, dev = ctx.M, w.device
        L = _lib.lib()
        with torch.cuda.device(dev):
            dl = dloss.reshape(-1).float()
            need_h, need_w = ctx.needs_input_grad[:2]
            dh = torch.empty((M, D), dtype=ctx.h_dtype, device=dev) if need_h else None
            dw = torch.empty((V, D), dtype=ctx.w_dtype, device=dev) if need_w else None
            nbytes = L.pnft_stream_xent_bwd_workspace_size(M, V, D)
            ws = _workspace(nbytes, dev)
            _lib.check(L.pnft_stream_xent_bwd(hc.data_ptr(), hc.shape[1], w.data_ptr(), _ld(w), saved.data_ptr(), dl.data_ptr(),
                                              dl.stride(0) if M > 1 else 1, ctx.reduction == "none", ctx.reduction == "mean",
                                              _ptr(dh), D, _DTYPES[ctx.h_dtype], _ptr(dw), D, _DTYPES[ctx.w_dtype],
                                              ws.data_ptr(), nbytes, M, V, D, _DTYPES[ctx.dt], _status_ptr(dev), _stream(dev)),
                       "pnft_stream_xent_bwd")
        return None if dh is None else dh.view(ctx.h_shape), dw, None, None, None, None, None, None


def streamed_cross_entropy(h: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100, *,
                           reduction: str = "mean", casts=None) -> torch.Tensor:
    """Cross entropy of the logits ``h @ weight.T`` against ``targets`` without keeping the
    logits (``F.cross_entropy``'s semantics, fp32 result): ``h`` ``[..., D]``, ``weight``
    ``[V, D]``, ``targets`` integer ids of ``h``'s leading shape. ``reduction``: ``"mean"`` over
    the rows whose target is not ``ignore_index``, ``"sum"``, or ``"none"`` (the rows' losses in
    ``targets``' shape, 0 where ignored; each row then has its own upstream gradient).

    Ignored rows cost nothing, and what they hold (NaN included) reaches no result: their
    gradient is 0. A target outside ``[0, V)`` that is not ``ignore_index`` gives a NaN loss
    and is reported by ``check_device_status()`` or the next call. ``casts``: an
    ``lm_ops.Bf16Casts`` with a current bf16 copy of ``weight``. Twice differentiating raises."""
    dev = _require_cuda("streamed_cross_entropy", h, weight, targets)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"streamed_cross_entropy: reduction {reduction!r}")
    if h.dim() == 0 or weight.dim() != 2 or h.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"streamed_cross_entropy: h {tuple(h.shape)}, weight {tuple(weight.shape)}: [..., D] and [V, D] expected")
    if 0 in weight.shape:
        raise RuntimeError(f"streamed_cross_entropy: empty weight {tuple(weight.shape)}")
    if targets.shape != h.shape[:-1]:
        raise RuntimeError(f"streamed_cross_entropy: targets {tuple(targets.shape)} for rows {tuple(h.shape[:-1])}")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise RuntimeError(f"streamed_cross_entropy: integer targets expected, got {targets.dtype}")
    for t in (h, weight):
        if t.dtype not in _DTYPES:
            raise RuntimeError(f"streamed_cross_entropy: float32, bfloat16 or float16 tensors expected, got {t.dtype}")
    dt = _compute_dtype(h, "streamed_cross_entropy")
    need = torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad)
    if targets.numel() == 0:  # as F.cross_entropy: nothing, 0, or 0 / 0; gradients of zeros
        zero = (h.float().sum() + weight.float().sum() * 0.0) if need else torch.zeros((), device=dev)
        if reduction == "none":
            return h.float().sum(-1)
        return zero * 0.0 if reduction == "sum" else zero * math.nan
    pre = casts.lookup(weight)[0] if casts is not None and dt == torch.bfloat16 and casts.lookup(weight) else None
    return _StreamXentFn.apply(h, weight, targets, int(ignore_index), reduction, dt, need, pre)


# ---------------------------------------------------------------- the block
def gated_mlp(x: torch.Tensor, gate: nn.Linear, up: nn.Linear, down: nn.Linear, activation: str = "silu", *,
              checkpoint_8bit: bool = False, casts=None) -> torch.Tensor:
    """``down(act(gate(x)) * up(x))`` (a SwiGLU / GEGLU feed-forward block) with ``gated_linear``;
    ``down`` is called as it is (an ``lm_ops.Linear`` brings its own weight gradient)."""
    h = gated_linear(x, gate.weight, up.weight, gate.bias, up.bias, activation, checkpoint_8bit=checkpoint_8bit, casts=casts)
    return down(h)
