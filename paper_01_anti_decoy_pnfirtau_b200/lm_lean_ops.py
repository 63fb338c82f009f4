"""Operators of a decoder's training step that can keep little for the backward pass,
on this library's tcgen05 kernels (csrc/gated.cu, csrc/xent_stream.cu, csrc/act8.cu
over the GEMM core csrc/gemm_tc.cuh). They stand beside ``mlp_gelu``,
``head_cross_entropy`` and ``Linear`` (lm_ops) of the Pre-LN decoder of the
reference's language-model experiments (experiments/exp4_wikitext2_lm.py:183-259).

- ``gated_linear``: ``act(x Wg^T + bg) * (x Wu^T + bu)`` (SwiGLU / GEGLU), both
  projections, the activation and the product in one kernel. Kept for the backward are x
  and, from width 896 on, where computing them again costs more, the two pre-activations
  with 24 bits each (as many bytes as a 16-bit composition keeps); with ``checkpoint_8bit``
  x in 8 bits alone. Calls of a few rows (single tokens) that need no gradient take the
  same entry.
- ``gated_mlp``: the block ``down(gated_linear(x))`` of three ``nn.Linear`` layers.
- ``streamed_cross_entropy``: the head's softmax cross entropy without its logits: kept
  are a 16-bit copy of the rows that count and 16 bytes a row beside it (room for all
  rows: ``2 M D + 16 M`` bytes), and the backward computes the logits again for one piece
  of the vocabulary at a time.
- ``act8_pack`` / ``act8_unpack`` / ``act8_weight_grad``: an activation in 8 bits (e4m3
  with a power of two per row and 128 columns) and the weight gradient that reads it (by
  way of a 16-bit copy in its workspace);
  ``lm_ops.Linear`` uses them when its ``checkpoint_8bit`` is set.

Operands are bfloat16 or float16: under CUDA autocast the inputs are cast to the
autocast dtype, else the input's dtype counts; float32 without autocast raises. CUDA
only; a CPU tensor raises. Results are bitwise reproducible on a given GPU. Forward-mode
tangents and tracing (``torch.jit.trace``, ``make_fx``) are refused; the ``act8_*`` calls
are not differentiable: their results require no gradient, whatever their inputs do.
"""
from __future__ import annotations

import math

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn as nn

from . import _lib
from .pnfirtau_ops import _DTYPES, _ptr, _raise, _require_cuda, _status_entry

_ACTS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}
_TYPES16 = (torch.bfloat16, torch.float16)


def _compute_dtype(x: torch.Tensor, what: str) -> torch.dtype:
    dt = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
    if dt not in _TYPES16:
        raise RuntimeError(f"{what}: bfloat16 or float16 expected (or CUDA autocast to one of them), got {dt}")
    return dt


def _plain_values(what: str, *tensors: torch.Tensor | None) -> None:
    """Raises where a call would lose what follows the values: the kernels write through addresses, so a tangent
    would vanish and a trace would hold an uninitialised buffer in the call's place."""
    if torch._C._get_tracing_state() is not None or (
            torch._C._len_torch_dispatch_stack() > 0
            and torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None):
        raise RuntimeError(f"{what}: cannot be traced")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what}: forward-mode differentiation is not available")


def _context(dev: torch.device) -> tuple[int, int]:
    """(status word's address, current stream) of ``dev``, which has to be the current
    device; raises if an earlier kernel on it has reported a failure."""
    w = _status_entry(dev)
    v = w.peek()
    if v != _lib.DEV_OK:
        w.reset()
        _raise(v, dev, "in an earlier call")
    return w.ptr, torch._C._cuda_getCurrentRawStream(dev.index)


def _elsewhere(dev: torch.device) -> bool:
    """``dev`` is not the current device (a call then runs under ``torch.cuda.device(dev)``)."""
    return torch._C._cuda_getDevice() != dev.index


def _new(rows: int, cols: int, dt: torch.dtype, dev: torch.device) -> torch.Tensor:
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dt, device=dev)  # cheaper to call than empty


def _bytes(n: int, dev: torch.device) -> torch.Tensor:
    return torch.empty_strided((n or 16,), (1,), dtype=torch.uint8, device=dev)


def _pad8(n: int) -> int:
    return (n + 7) // 8 * 8


def _ld(t: torch.Tensor) -> int:
    """Row stride of a matrix; a single row's is free, so its padded width."""
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else (cols + 7) // 8 * 8


def _unit_rows(t: torch.Tensor, dt: torch.dtype) -> torch.Tensor:
    """``t`` (2-D) in ``dt`` with unit column stride and rows that do not overlap."""
    if t.dtype is dt:
        ld, unit = t.stride()
        if unit == 1 and ld >= t.shape[1]:
            return t
    if t.dtype != dt:
        t = t.to(dt)
    rows, cols = t.shape
    return t if (t.stride(1) == 1 or cols == 1) and (rows <= 1 or t.stride(0) >= cols) else t.contiguous()


def _rows16(t: torch.Tensor, dt: torch.dtype) -> torch.Tensor:
    """``t`` (2-D) in ``dt`` as rows that a TMA map takes: unit column stride, row stride
    a multiple of 8 elements, 16-byte base. A view of ``t`` when it is that already."""
    if t.dtype is dt and t.data_ptr() % 16 == 0:
        ld, unit = t.stride()
        if unit == 1 and ld % 8 == 0 and ld >= t.shape[1]:
            return t
    t = _unit_rows(t, dt)
    if t.data_ptr() % 16 == 0 and _ld(t) % 8 == 0:
        return t
    rows, cols = t.shape
    out = _new(rows, _pad8(cols), dt, t.device)[:, :cols]
    rc = _lib.lib().pnft_copy_rows16(t.data_ptr(), _ld(t), out.data_ptr(), _pad8(cols), rows, cols, _context(t.device)[1])
    _lib.check(rc, "pnft_copy_rows16")
    return out


# ---------------------------------------------------------------- 8-bit activations
def _act8_row_bytes(D: int) -> int:
    return (D + 15) // 16 * 16 + ((D + 127) // 128 + 15) // 16 * 16


class Act8:
    """An activation in 8 bits: ``data`` holds a row's e4m3 bytes (padded to a multiple of
    16) and behind them one int8 exponent per block of 128 columns; an element's value is
    ``e4m3 * 2^exponent``. ``shape`` and ``dtype`` are the packed tensor's."""

    __slots__ = ("data", "shape", "dtype")

    def __init__(self, data: torch.Tensor, shape: torch.Size, dtype: torch.dtype):
        self.data, self.shape, self.dtype = data, shape, dtype

    @property
    def width(self) -> int:
        return self.shape[-1]

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def _layout(self):
        """(bytes' address, row stride, exponents' address, row stride, rows, columns), once the
        buffer is known to hold what ``shape`` says."""
        data, shape = self.data, self.shape
        n = len(shape)
        D = shape[-1] if n else 0
        rows = shape[0] if n == 2 else math.prod(shape[:-1])
        ld, at = _act8_row_bytes(D), data.data_ptr()
        if (D == 0 or data.shape != (rows, ld) or data.dtype is not torch.uint8 or not data.is_contiguous() or at % 16
                or self.dtype not in _DTYPES):
            raise RuntimeError(f"Act8: {data.dtype} buffer {tuple(data.shape)} with strides {data.stride()} does not hold "
                               f"{tuple(shape)} of {self.dtype} in 8 bits")
        return at, ld, at + (D + 15) // 16 * 16, ld, rows, D


def act8_pack(x: torch.Tensor) -> Act8:
    """``x`` (float32, bfloat16 or float16; ``[..., D]``) in 8 bits: per row and block of
    128 columns e4m3 values times the least power of two that brings the block's largest
    magnitude to 448 or less, rounded to nearest even. NaN and infinities become NaN. The
    powers reach from 2^-110 to 2^120 (float16: 2^-15 to 2^8), so blocks below 2^-110 keep
    fewer bits, and in the largest one magnitudes end at 240 times it."""
    dev = _require_cuda("act8_pack", x)
    _plain_values("act8_pack", x)
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise RuntimeError(f"act8_pack: float32, bfloat16 or float16 expected, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise RuntimeError(f"act8_pack: rows of at least one column expected, got {tuple(x.shape)}")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return act8_pack(x)
    shape = x.shape
    D = shape[-1]
    x2 = _unit_rows(x if x.dim() == 2 else x.reshape(-1, D), x.dtype)
    M = x2.shape[0]
    ld = _act8_row_bytes(D)
    data = _new(M, ld, torch.uint8, dev)
    q = data.data_ptr()
    rc = _lib.lib().pnft_act8_pack(x2.data_ptr(), x2.stride(0) if M > 1 else D, q, ld, q + (D + 15) // 16 * 16, ld, M, D, code,
                                   _context(dev)[1])
    _lib.check(rc, "pnft_act8_pack")
    return Act8(data, shape, x.dtype)


def _act8_rows(p: Act8, dt: torch.dtype, width: int) -> torch.Tensor:
    """The values as rows of ``width`` columns of ``dt`` (those past ``p.width`` undefined)."""
    q, ldq, e, lde, M, D = p._layout()
    dev = p.data.device
    y = _new(M, width, dt, dev)
    rc = _lib.lib().pnft_act8_unpack(q, ldq, e, lde, y.data_ptr(), width, M, D, _DTYPES[dt], _context(dev)[1])
    _lib.check(rc, "pnft_act8_unpack")
    return y


def act8_unpack(p: Act8) -> torch.Tensor:
    """The tensor that ``p`` stands for, in the shape and dtype that were packed (exact:
    the dtype holds every packed value)."""
    dev = _require_cuda("act8_unpack", p.data)
    _plain_values("act8_unpack", p.data)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return act8_unpack(p)
    y = _act8_rows(p, p.dtype, p.width)
    return y if y.shape == p.shape else y.view(p.shape)


def act8_weight_grad(dy: torch.Tensor, p: Act8, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``dy^T x`` for the packed ``x``: the weight gradient ``[N, D]`` of a Linear layer
    from its output's gradient ``dy`` (``[..., N]``, bfloat16 or float16, as many rows as
    ``x``) and its input kept in 8 bits; fp32 sums."""
    dev = _require_cuda("act8_weight_grad", dy, p.data)
    _plain_values("act8_weight_grad", dy)
    if dy.dtype not in _TYPES16 or out_dtype not in _DTYPES:
        raise RuntimeError(f"act8_weight_grad: bfloat16 or float16 gradient and a float32, bfloat16 or float16 result expected, "
                           f"got {dy.dtype} and {out_dtype}")
    if dy.dtype == torch.float16 and p.dtype != torch.float16:
        raise RuntimeError(f"act8_weight_grad: a float16 gradient needs a float16 activation, got {p.dtype}")
    if dy.dim() == 0 or dy.shape[-1] == 0:
        raise RuntimeError(f"act8_weight_grad: rows of at least one column expected, got {tuple(dy.shape)}")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return act8_weight_grad(dy, p, out_dtype)
    q, ldq, e, lde, M, D = p._layout()
    N = dy.shape[-1]
    dy2 = dy if dy.dim() == 2 else dy.reshape(-1, N)
    if dy2.shape[0] != M:
        raise RuntimeError(f"act8_weight_grad: {dy2.shape[0]} rows of gradient but {M} of activation")
    dy2 = _rows16(dy2, dy.dtype) if N % 8 == 0 else _unit_rows(dy2, dy.dtype)
    dw = _new(N, D, out_dtype, dev)
    L = _lib.lib()
    nbytes = L.pnft_act8_weight_grad_workspace_size(M, N, D)
    ws = _bytes(nbytes, dev)
    status, stream = _context(dev)
    rc = L.pnft_act8_weight_grad(dy2.data_ptr(), _ld(dy2), q, ldq, e, lde, dw.data_ptr(), D, _DTYPES[out_dtype], ws.data_ptr(),
                                 nbytes, M, N, D, _DTYPES[dy.dtype], status, stream)
    _lib.check(rc, "pnft_act8_weight_grad")
    return dw


# ---------------------------------------------------------------- gated product
# From this input width on the forward keeps the pre-activations (6 bytes of each pair,
# written once and read once by a pointwise backward kernel); below it the backward
# computes them again, which costs 4 M D F operations but no memory traffic. Forward and
# backward on a B200 (bf16, 16384 rows, F = 4 D), kept against computed again: D = 512
# 286 and 249 us, 768 503 and 480, 1024 820 and 840, 2048 2700 and 3102.
_KEEP_FROM = 896
# Rows up to which a call that keeps nothing leaves unaligned rows as they are: all that the few-row
# kernel takes where the width is no multiple of 8, since aligned copies gain no vector loads there
# (B200, 32 rows from cold L2, copied against in place: 1001 x 4096 35 and 22 us, 2047 x 5461 115
# and 57); fewer where they do (2-byte aligned views, 1024 x 4096 27 and 25, 4096 x 16384 210 and 270).
_FEW_VECTOR = 24


def _gated_forward(x, wg, wu, bg, bu, act: int, dt: torch.dtype, keep: bool):
    """(h, x's rows, the weights' rows, the kept pre-activations or None)."""
    dev = x.device
    F_, D = wg.shape
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, D)
    M = x2.shape[0]
    few = _lib.GATED_FEW_ROWS if D % 8 else _FEW_VECTOR
    rows = _rows16 if keep or M > few else _unit_rows
    x2, wg, wu = rows(x2, dt), rows(wg, dt), rows(wu, dt)
    h = _new(M, F_, dt, dev)
    pre = _new(3 * M, _pad8(F_), torch.int16, dev) if keep else None
    b = bg if bg is not None else bu
    status, stream = _context(dev)
    rc = _lib.lib().pnft_gated_fwd(
        x2.data_ptr(), _ld(x2), wg.data_ptr(), _ld(wg), wu.data_ptr(), _ld(wu), _ptr(bg), _ptr(bu),
        _lib.DTYPE_F32 if b is None else _DTYPES[b.dtype], h.data_ptr(), F_, _ptr(pre), _pad8(F_), M, D, F_, act, _DTYPES[dt],
        status, stream)
    _lib.check(rc, "pnft_gated_fwd")
    return h if flat else h.view(*x.shape[:-1], F_), x2, wg, wu, pre


class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, bg, bu, act: int, dt: torch.dtype, in8: bool, copies):
        wgc, wuc = copies if copies is not None else (wg, wu)
        h, x2, wgc, wuc, pre = _gated_forward(x, wgc, wuc, bg, bu, act, dt, not in8 and wg.shape[1] >= _KEEP_FROM)
        ctx.act8 = None
        if in8:
            p = act8_pack(x2)
            x2, ctx.act8 = p.data, (p.shape, p.dtype)
        ctx.save_for_backward(x2, pre, wgc, wuc, bg, bu)
        ctx.meta = (act, dt, x.shape, x.dtype, wg.dtype)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        dev = dh.device
        if _elsewhere(dev):
            with torch.cuda.device(dev):
                return _gated_backward(ctx, dh)
        return _gated_backward(ctx, dh)


def _gated_backward(ctx, dh):
    x2, pre, wg, wu, bg, bu = ctx.saved_tensors
    act, dt, x_shape, x_dtype, w_dtype = ctx.meta
    dev = wg.device
    F_, D = wg.shape
    nx, nwg, nwu, nbg, nbu = ctx.needs_input_grad[:5]
    if ctx.act8 is not None:
        x2 = _act8_rows(Act8(x2, *ctx.act8), dt, _pad8(D))
        ldx = _pad8(D)
    else:
        x2 = _rows16(x2, dt)  # a copy only where a forward of few rows took them as they were
        ldx = _ld(x2)
    wg, wu = _rows16(wg, dt), _rows16(wu, dt)
    M = x2.shape[0]
    dh = dh.reshape(-1, F_)
    dh = _rows16(dh, dt) if F_ % 8 == 0 else _unit_rows(dh, dt)
    dx = _new(M, D, x_dtype, dev) if nx else None
    dwg = _new(F_, D, w_dtype, dev) if nwg else None
    dwu = _new(F_, D, w_dtype, dev) if nwu else None
    b = bg if bg is not None else bu
    b_dtype = torch.float32 if b is None else b.dtype
    dbg = torch.empty(F_, dtype=b_dtype, device=dev) if nbg and bg is not None else None
    dbu = torch.empty(F_, dtype=b_dtype, device=dev) if nbu and bu is not None else None
    L = _lib.lib()
    nbytes = L.pnft_gated_bwd_workspace_size(M, D, F_)
    ws = _bytes(nbytes, dev)
    status, stream = _context(dev)
    rc = L.pnft_gated_bwd(
        x2.data_ptr(), ldx, wg.data_ptr(), _ld(wg), wu.data_ptr(), _ld(wu), _ptr(bg), _ptr(bu), _DTYPES[b_dtype], _ptr(pre),
        _pad8(F_), dh.data_ptr(), _ld(dh), _ptr(dx), D, _DTYPES[x_dtype], _ptr(dwg), _ptr(dwu), D, _DTYPES[w_dtype], _ptr(dbg),
        _ptr(dbu), ws.data_ptr(), nbytes, M, D, F_, act, _DTYPES[dt], status, stream)
    _lib.check(rc, "pnft_gated_bwd")
    if nx and len(x_shape) != 2:
        dx = dx.view(x_shape)
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
    bf16 copies of the weights, used when the dtype is bf16.

    The gradients of the pre-activations are rounded to the 16-bit type before the products
    with the weights and x. In float16 they overflow past 65504 as in a float16 composition:
    scale the loss accordingly."""
    biases = () if b_gate is None and b_up is None else tuple(b for b in (b_gate, b_up) if b is not None)
    dev = _require_cuda("gated_linear", x, w_gate, w_up, *biases)
    _plain_values("gated_linear", x, w_gate, w_up, *biases)
    act = _ACTS.get(activation)
    if act is None:
        raise ValueError(f"gated_linear: activation {activation!r} (one of {sorted(_ACTS)})")
    if x.dim() == 0 or w_gate.dim() != 2 or w_gate.shape != w_up.shape or x.shape[-1] != w_gate.shape[1]:
        raise RuntimeError(f"gated_linear: x {tuple(x.shape)}, weights {tuple(w_gate.shape)} and {tuple(w_up.shape)}: [..., D] "
                           "and twice [F, D] expected")
    if 0 in w_gate.shape:
        raise RuntimeError(f"gated_linear: empty weights {tuple(w_gate.shape)}")
    for b in biases:
        if b.shape != w_gate.shape[:1]:
            raise RuntimeError(f"gated_linear: bias {tuple(b.shape)} for {w_gate.shape[0]} columns")
        if b.dtype not in _DTYPES or b.dtype != biases[0].dtype:
            raise RuntimeError("gated_linear: float32, bfloat16 or float16 biases of one dtype expected")
    if x.dtype not in _DTYPES or w_gate.dtype not in _DTYPES or w_up.dtype != w_gate.dtype:
        raise RuntimeError(f"gated_linear: float32, bfloat16 or float16 tensors and weights of one dtype expected, got {x.dtype}, "
                           f"{w_gate.dtype} and {w_up.dtype}")
    dt = _compute_dtype(x, "gated_linear")
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return gated_linear(x, w_gate, w_up, b_gate, b_up, activation, checkpoint_8bit=checkpoint_8bit, casts=casts)
    if biases:
        b_gate, b_up = (None if b is None else b.contiguous() for b in (b_gate, b_up))
    copies = casts.lookup(w_gate, w_up) if casts is not None and dt == torch.bfloat16 else None
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or any(b.requires_grad for b in biases)):
        return _GatedLinearFn.apply(x, w_gate, w_up, b_gate, b_up, act, dt, checkpoint_8bit, copies)
    wg, wu = copies if copies is not None else (w_gate, w_up)
    return _gated_forward(x, wg, wu, b_gate, b_up, act, dt, False)[0]


# ---------------------------------------------------------------- streamed cross entropy
def _xent_forward(h, weight, targets, ignore_index: int, reduction: str, dt: torch.dtype, save: bool):
    """(loss, the kept state or None, the weight's rows)."""
    dev = h.device
    V, D = weight.shape
    h2 = _unit_rows(h if h.dim() == 2 else h.reshape(-1, D), dt)
    M = h2.shape[0]
    w = _rows16(weight, dt) if save or M > _lib.XENT_FEW_ROWS else _unit_rows(weight, dt)
    t = targets if targets.dim() == 1 else targets.reshape(-1)
    if t.dtype != torch.int64 or not t.is_contiguous():
        t = t.to(torch.int64).contiguous()
    L = _lib.lib()
    per_row = reduction == "none"
    loss = torch.empty(targets.shape if per_row else (), dtype=torch.float32, device=dev)
    at = loss.data_ptr()
    saved = _bytes(L.pnft_stream_xent_saved_size(M, D), dev) if save else None
    nbytes = L.pnft_stream_xent_fwd_workspace_size(M, V, D, save)
    ws = _bytes(nbytes, dev)
    status, stream = _context(dev)
    rc = L.pnft_stream_xent_fwd(h2.data_ptr(), h2.stride(0) if M > 1 else D, w.data_ptr(), _ld(w), t.data_ptr(), ignore_index,
                                _ptr(saved), at if per_row else None, None if per_row else at, reduction == "mean",
                                ws.data_ptr(), nbytes, M, V, D, _DTYPES[dt], status, stream)
    _lib.check(rc, "pnft_stream_xent_fwd")
    return loss, saved, w


class _StreamXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, targets, ignore_index: int, reduction: str, dt: torch.dtype, copy):
        loss, saved, w = _xent_forward(h, weight if copy is None else copy, targets, ignore_index, reduction, dt, True)
        ctx.save_for_backward(saved, w)
        ctx.meta = (targets.numel(), dt, reduction, h.shape, h.dtype, weight.dtype)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        if _elsewhere(dloss.device):
            with torch.cuda.device(dloss.device):
                return _xent_backward(ctx, dloss)
        return _xent_backward(ctx, dloss)


def _xent_backward(ctx, dloss):
    saved, w = ctx.saved_tensors
    M, dt, reduction, h_shape, h_dtype, w_dtype = ctx.meta
    w = _rows16(w, dt)  # a copy only where a hook brought the saved rows back without their padding
    V, D = w.shape
    dev = w.device
    L = _lib.lib()
    per_row = reduction == "none"
    if per_row:
        dloss = dloss.reshape(-1)
    dh = _new(M, D, h_dtype, dev) if ctx.needs_input_grad[0] else None
    dw = _new(V, D, w_dtype, dev) if ctx.needs_input_grad[1] else None
    nbytes = L.pnft_stream_xent_bwd_workspace_size(M, V, D)
    ws = _bytes(nbytes, dev)
    status, stream = _context(dev)
    rc = L.pnft_stream_xent_bwd(w.data_ptr(), _ld(w), saved.data_ptr(), dloss.data_ptr(), dloss.stride(0) if per_row else 1,
                                per_row, reduction == "mean", _ptr(dh), D, _DTYPES[h_dtype], _ptr(dw), D, _DTYPES[w_dtype],
                                ws.data_ptr(), nbytes, M, V, D, _DTYPES[dt], status, stream)
    _lib.check(rc, "pnft_stream_xent_bwd")
    if dh is not None and len(h_shape) != 2:
        dh = dh.view(h_shape)
    return dh, dw, None, None, None, None, None


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
    ``lm_ops.Bf16Casts`` with a current bf16 copy of ``weight``. Twice differentiating raises.

    Logits are fp32 and so are the exponents that come from them: a probability in the gradient
    is off by about 2^-24 times the largest logit's magnitude, and logits past 2^30 have no
    result. The logits' gradient is rounded to the 16-bit type, in float16 scaled by one factor
    for all rows: with ``reduction="none"`` a row whose upstream gradient is far below the
    largest keeps fewer bits of its small probabilities."""
    dev = _require_cuda("streamed_cross_entropy", h, weight, targets)
    _plain_values("streamed_cross_entropy", h, weight)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"streamed_cross_entropy: reduction {reduction!r}")
    if h.dim() == 0 or weight.dim() != 2 or h.shape[-1] != weight.shape[1]:
        raise RuntimeError(f"streamed_cross_entropy: h {tuple(h.shape)}, weight {tuple(weight.shape)}: [..., D] and [V, D] expected")
    if weight.numel() == 0:
        raise RuntimeError(f"streamed_cross_entropy: empty weight {tuple(weight.shape)}")
    if targets.shape != h.shape[:-1]:
        raise RuntimeError(f"streamed_cross_entropy: targets {tuple(targets.shape)} for rows {tuple(h.shape[:-1])}")
    if targets.dtype not in (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8):
        raise RuntimeError(f"streamed_cross_entropy: integer targets expected, got {targets.dtype}")
    if h.dtype not in _DTYPES or weight.dtype not in _DTYPES:
        raise RuntimeError(f"streamed_cross_entropy: float32, bfloat16 or float16 tensors expected, got {h.dtype} and {weight.dtype}")
    dt = _compute_dtype(h, "streamed_cross_entropy")
    if targets.numel() == 0:  # as F.cross_entropy: nothing, 0, or 0 / 0; gradients of zeros
        zero = (h.float().sum(-1) if reduction == "none" else h.float().sum()) + weight[:0].float().sum()
        return zero * math.nan if reduction == "mean" else zero
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return streamed_cross_entropy(h, weight, targets, ignore_index, reduction=reduction, casts=casts)
    copy = casts.lookup(weight) if casts is not None and dt == torch.bfloat16 else None
    copy = None if copy is None else copy[0]
    if torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad):
        return _StreamXentFn.apply(h, weight, targets, int(ignore_index), reduction, dt, copy)
    return _xent_forward(h, weight if copy is None else copy, targets, int(ignore_index), reduction, dt, False)[0]


# ---------------------------------------------------------------- the block
def gated_mlp(x: torch.Tensor, gate: nn.Linear, up: nn.Linear, down: nn.Linear, activation: str = "silu", *,
              checkpoint_8bit: bool = False, casts=None) -> torch.Tensor:
    """``down(act(gate(x)) * up(x))`` (a SwiGLU / GEGLU feed-forward block) with ``gated_linear``;
    ``down`` is called as it is (an ``lm_ops.Linear`` brings its own weight gradient)."""
    h = gated_linear(x, gate.weight, up.weight, gate.bias, up.bias, activation, checkpoint_8bit=checkpoint_8bit, casts=casts)
    return down(h)
