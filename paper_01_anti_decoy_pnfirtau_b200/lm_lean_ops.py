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

import contextlib
import math
from dataclasses import dataclass

import torch
import torch.nn as nn

from . import _lib
from .pnfirtau_ops import _DTYPES, _check_pending, _ptr, _require_cuda, _status_ptr

_ACTS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
_TYPES16 = (torch.bfloat16, torch.float16)


def _compute_dtype(x: torch.Tensor, what: str) -> torch.dtype:
    dt = torch.get_autocast_dtype("cuda") if x.is_cuda and torch.is_autocast_enabled("cuda") else x.dtype
    if dt not in _TYPES16:
        raise RuntimeError(f"{what}: bfloat16 or float16 expected (or CUDA autocast to one of them), got {dt}")
    return dt


_HERE = contextlib.nullcontext()


def _on(dev: torch.device):
    """Makes ``dev`` the current device, as the library's launches need (free when it is)."""
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(dev.index)


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
    with _on(dev):
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
    with _on(p.q.device):
        return _act8_rows(p, p.dtype).reshape(p.shape)


def act8_weight_grad(dy: torch.Tensor, p: Act8, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``dy^T x`` for the packed ``x``: the weight gradient ``[N, D]`` of a Linear layer
    from its output's gradient ``dy`` (``[..., N]``, bfloat16 or float16, as many rows as
    ``x``) and its input kept in 8 bits; fp32 sums."""
    dev = _require_cuda("act8_weight_grad", dy, p.q)
    if out_dtype not in _DTYPES:
        raise RuntimeError(f"act8_weight_grad: float32, bfloat16 or float16 result expected, got {out_dtype}")
    if dy.dtype not in _TYPES16:
        raise RuntimeError(f"act8_weight_grad: bfloat16 or float16 gradient expected, got {dy.dtype}")
    if dy.dtype == torch.float16 and p.dtype != torch.float16:
        raise RuntimeError(f"act8_weight_grad: a float16 gradient needs a float16 activation, got {p.dtype}")
    if dy.dim() == 0 or dy.shape[-1] == 0:
        raise RuntimeError(f"act8_weight_grad: rows of at least one column expected, got {tuple(dy.shape)}")
    dy2 = dy.detach().reshape(-1, dy.shape[-1])
    if dy2.shape[0] != p.q.shape[0]:
        raise RuntimeError(f"act8_weight_grad: {dy2.shape[0]} rows of gradient but {p.q.shape[0]} of activation")
    with _on(dev):
        return _weight_grad(_rows16(dy2, dy.dtype), _act8_rows(p, dy.dtype), out_dtype)


def _weight_grad(dy: torch.Tensor, x: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    """``dy^T x`` of two ``_rows16`` matrices."""
    K, M = dy.shape
    N, dev = x.shape[1], dy.device
    out = torch.empty((M, N), dtype=out_dtype, device=dev)
    L = _lib.lib()
    nbytes = L.pnft_weight_grad_workspace_size(K, M, N)
    ws = _workspace(nbytes, dev)
    rc = L.pnft_weight_grad(dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), out.data_ptr(), None, N, M, M, _DTYPES[out_dtype],
                            ws.data_ptr(), nbytes, K, M, N, _DTYPES[dy.dtype], _status_ptr(dev), _stream(dev))
    _lib.check(rc, "pnft_weight_grad")
    return out


# ---------------------------------------------------------------- gated product
# From this input width on the forward keeps the pre-activations (6 bytes per element of each,
# written once and read once) and the backward reads them; below it computes them again, which
# costs 4 M D F operations but no memory. <measured below>
_KEEP_FROM = 640


def _gated_forward(x, wg, wu, bg, bu, act: int, dt: torch.dtype, keep: bool):
    """(h, x's rows, the weights' rows, the kept pre-activations or None)."""
    dev = x.device
    _check_pending(dev)
    F_, D = wg.shape
    with _on(dev):
        x2 = _rows16(x.reshape(-1, D), dt)
        wgc, wuc = _rows16(wg, dt), _rows16(wu, dt)
        M = x2.shape[0]
        h = torch.empty((M, F_), dtype=dt, device=dev)
        pre = torch.empty((3, M, _pad8(F_)), dtype=torch.int16, device=dev) if keep else None
        b = bg if bg is not None else bu
        rc = _lib.lib().pnft_gated_fwd(
            x2.data_ptr(), _ld(x2), wgc.data_ptr(), _ld(wgc), wuc.data_ptr(), _ld(wuc), _ptr(bg), _ptr(bu),
            _lib.DTYPE_F32 if b is None else _DTYPES[b.dtype], h.data_ptr(), F_, _ptr(pre), _pad8(F_), M, D, F_, act,
            _DTYPES[dt], _status_ptr(dev), _stream(dev))
        _lib.check(rc, "pnft_gated_fwd")
    return h.view(*x.shape[:-1], F_), x2, wgc, wuc, pre


class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act: int, dt: torch.dtype, in8: bool, copies):
        wgc, wuc = copies if copies is not None else (wg, wu)
        h, x2, wgc, wuc, pre = _gated_forward(x, wgc, wuc, bg, bu, act, dt, not in8 and wg.shape[1] >= _KEEP_FROM)
        p = act8_pack(x2) if in8 else None
        if in8:
            ctx.save_for_backward(p.q, p.exponents, wgc, wuc, bg, bu)
        else:
            ctx.save_for_backward(x2, pre, wgc, wuc, bg, bu)
        ctx.p8 = (p.shape, p.dtype) if in8 else None
        ctx.act, ctx.dt, ctx.x_shape, ctx.x_dtype, ctx.w_dtype = act, dt, x.shape, x.dtype, wg.dtype
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        a, b, wg, wu, bg, bu = ctx.saved_tensors
        dt, dev = ctx.dt, wg.device
        F_, D = wg.shape
        need = ctx.needs_input_grad
        L = _lib.lib()
        with _on(dev):
            x2, pre = (a, b) if ctx.p8 is None else (_act8_rows(Act8(a, b, *ctx.p8), dt), None)
            M = x2.shape[0]
            dh2 = dh.reshape(-1, F_)
            if dh2.dtype != dt:
                dh2 = dh2.to(dt)
            if F_ % 8 == 0:
                dh2 = _rows16(dh2, dt)
            elif dh2.stride(1) != 1 or dh2.stride(0) < F_:
                dh2 = dh2.contiguous()
            grad = lambda n, shape, t: torch.empty(shape, dtype=t, device=dev) if n else None  # noqa: E731
            dx = grad(need[0], ctx.x_shape, ctx.x_dtype)
            dwg, dwu = grad(need[1], (F_, D), ctx.w_dtype), grad(need[2], (F_, D), ctx.w_dtype)
            bias = bg if bg is not None else bu
            b_dtype = torch.float32 if bias is None else bias.dtype
            dbg, dbu = grad(bg is not None and need[3], F_, b_dtype), grad(bu is not None and need[4], F_, b_dtype)
            nbytes = L.pnft_gated_bwd_workspace_size(M, D, F_)
            ws = _workspace(nbytes, dev)
            rc = L.pnft_gated_bwd(
                x2.data_ptr(), _ld(x2), wg.data_ptr(), _ld(wg), wu.data_ptr(), _ld(wu), _ptr(bg), _ptr(bu), _DTYPES[b_dtype],
                _ptr(pre), _pad8(F_), dh2.data_ptr(), max(_ld(dh2) if F_ % 8 == 0 else dh2.stride(0), F_), _ptr(dx), D,
                _DTYPES[ctx.x_dtype], _ptr(dwg), _ptr(dwu), D, _DTYPES[ctx.w_dtype], _ptr(dbg), _ptr(dbu), ws.data_ptr(),
                nbytes, M, D, F_, ctx.act, _DTYPES[dt], _status_ptr(dev), _stream(dev))
            _lib.check(rc, "pnft_gated_bwd")
        return dx, dwg, dwu, dbg, dbu, None, None, None, None


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
    copies = casts.lookup(w_gate, w_up) if casts is not None and dt == torch.bfloat16 else None
    if torch.is_grad_enabled() and any(t.requires_grad for t in ts):
        return _GatedLinearFn.apply(x, w_gate, w_up, b_gate, b_up, _ACTS[activation], dt, checkpoint_8bit, copies)
    wg, wu = copies if copies is not None else (w_gate, w_up)
    return _gated_forward(x, wg, wu, b_gate, b_up, _ACTS[activation], dt, False)[0]


# ---------------------------------------------------------------- streamed cross entropy
def _xent_forward(h, weight, targets, ignore_index: int, reduction: str, dt: torch.dtype):
    """(loss, the rows that count, the kept state, the weight's rows)."""
    dev = h.device
    _check_pending(dev)
    V, D = weight.shape
    L = _lib.lib()
    with _on(dev):
        h2 = h.reshape(-1, D)
        if h2.dtype != dt:
            h2 = h2.to(dt)
        if h2.stride(1) != 1 and D > 1 or h2.stride(0) < D:
            h2 = h2.contiguous()
        w = _rows16(weight, dt)
        t = targets.reshape(-1)
        if t.dtype != torch.int64 or not t.is_contiguous():
            t = t.to(torch.int64).contiguous()
        M, Dp = h2.shape[0], _pad8(D)
        hc = torch.empty(((M + 127) // 128 * 128, Dp), dtype=dt, device=dev)
        saved = _workspace(L.pnft_stream_xent_saved_size(M), dev)
        rows = torch.empty(M, dtype=torch.float32, device=dev) if reduction == "none" else None
        loss = torch.empty((), dtype=torch.float32, device=dev) if rows is None else None
        nbytes = L.pnft_stream_xent_fwd_workspace_size(M, V)
        ws = _workspace(nbytes, dev)
        rc = L.pnft_stream_xent_fwd(h2.data_ptr(), h2.stride(0), w.data_ptr(), _ld(w), t.data_ptr(), ignore_index,
                                    hc.data_ptr(), Dp, saved.data_ptr(), _ptr(rows), _ptr(loss), reduction == "mean",
                                    ws.data_ptr(), nbytes, M, V, D, _DTYPES[dt], _status_ptr(dev), _stream(dev))
        _lib.check(rc, "pnft_stream_xent_fwd")
    return (loss if rows is None else rows.view(targets.shape)), hc, saved, w


class _StreamXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, targets, ignore_index: int, reduction: str, dt: torch.dtype, copy):
        loss, hc, saved, w = _xent_forward(h, weight if copy is None else copy, targets, ignore_index, reduction, dt)
        ctx.save_for_backward(hc, saved, w)
        ctx.M, ctx.dt, ctx.reduction = targets.numel(), dt, reduction
        ctx.h_shape, ctx.h_dtype, ctx.w_dtype = h.shape, h.dtype, weight.dtype
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        hc, saved, w = ctx.saved_tensors
        V, D = w.shape
        M, dev = ctx.M, w.device
        L = _lib.lib()
        with _on(dev):
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
        return None if dh is None else dh.view(ctx.h_shape), dw, None, None, None, None, None


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
    copy = casts.lookup(weight) if casts is not None and dt == torch.bfloat16 else None
    copy = None if copy is None else copy[0]
    if need:
        return _StreamXentFn.apply(h, weight, targets, int(ignore_index), reduction, dt, copy)
    return _xent_forward(h, weight if copy is None else copy, targets, int(ignore_index), reduction, dt)[0]


# ---------------------------------------------------------------- the block
def gated_mlp(x: torch.Tensor, gate: nn.Linear, up: nn.Linear, down: nn.Linear, activation: str = "silu", *,
              checkpoint_8bit: bool = False, casts=None) -> torch.Tensor:
    """``down(act(gate(x)) * up(x))`` (a SwiGLU / GEGLU feed-forward block) with ``gated_linear``;
    ``down`` is called as it is (an ``lm_ops.Linear`` brings its own weight gradient)."""
    h = gated_linear(x, gate.weight, up.weight, gate.bias, up.bias, activation, checkpoint_8bit=checkpoint_8bit, casts=casts)
    return down(h)
