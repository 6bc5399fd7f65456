"""Operators of a transformer block beside ``linear``, ``layer_norm`` and ``attention`` of ``torch_ops``: the RMS norm of a residual
stream (with an 8-bit output for serving), 8-bit quantisation of rows, rotary positions with several axes, and the linear layer with
activation and residual in its epilogue, in 16 and in 8 bits.

They are ``torch.ops.mvit.*`` operators like those, with fake (meta) implementations and autograd formulas on the backward kernels; the
functions below are their entry points, re-exported by ``torch_ops``.  CUDA (ROCm) tensors only.  16-bit operands are bf16 or fp16 as
the tensors are (fp16 runs in libmiphei_hip_f16.so), never a mixture; the work goes to the tensors' device, on its current stream.

Registered through ``torch.library.Library`` and an ``autograd.Function`` instead of ``torch.library.custom_op``: the same operators at
5 against 15 us of host time a call, and 51 against 84 us for a forward and backward (measured on the host alone), which is what a call
on one token costs.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Sequence

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import ops

_LIB = torch.library.Library("mvit", "FRAGMENT")
_HALF = (torch.bfloat16, torch.float16)
_E4M3 = torch.float8_e4m3fn
_ROWS_MAX = 2 ** 31 - 1


def _define(schema, impl, fake, function=None):
    """The operator `schema` with its GPU implementation, its fake one and, where it has gradients, its autograd.Function."""
    name = schema.split("(", 1)[0]
    _LIB.define(schema)
    _LIB.impl(name, impl, "CUDA")
    torch.library.register_fake(f"mvit::{name}", fake, lib=_LIB)
    op = getattr(torch.ops.mvit, name).default
    if function is not None:
        def autograd(*args):
            if torch.is_grad_enabled() and any(isinstance(a, Tensor) and a.requires_grad for a in args):
                return function.apply(*args)
            with torch._C._AutoDispatchBelowAutograd():
                return op(*args)
        _LIB.impl(name, autograd, "AutogradCUDA")
    return op


def _bad(op, why):
    return ValueError(f"mvit::{op}: {why}")


def _same_place(op, x, *others):
    for t in others:
        if t is not None and t.device != x.device:
            raise _bad(op, f"tensors on {x.device} and {t.device}")


def _half_type(op, *tensors):
    """The one 16-bit type among the operands (None: all f32); a mixture is refused, and so is any type but bf16, fp16 and f32."""
    half = None
    for t in tensors:
        d = t.dtype if isinstance(t, Tensor) else t
        if d is None or d == torch.float32:
            continue
        if d not in _HALF:
            raise _bad(op, f"operands are bfloat16, float16 or float32, got {d}")
        if half is not None and d != half:
            raise _bad(op, "bfloat16 and float16 operands in one call")
        half = d
    return half


def _no_grad(op, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"mvit::{op} has no gradient: call it under torch.no_grad() or on detached tensors")


def _launch(fn, device, half, *args, **kw):
    """fn on `device`'s current stream, in the library of the 16-bit type `half` (None: either)."""
    mode = "f16" if half == torch.float16 else "bf16"
    here = device.index is None or device.index == torch.cuda.current_device()
    if here and (half is None or L.operand_mode() == mode):
        return fn(*args, **kw)
    with contextlib.ExitStack() as stack:
        if not here:
            stack.enter_context(torch.cuda.device(device))
        if half is not None:
            stack.enter_context(L.operands(mode))
        return fn(*args, **kw)


def _rows(t):
    """[rows, last] view of t whose rows are dense (any row stride of at least their length), a copy only where there is none."""
    D = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, D)
    if (D > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < D):
        t = t.contiguous()
    return t


# ------------------------------------------------------------------ RMS norm with the residual's addition
def _norm_check(op, x, residual, weight, out=None):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 16384:
        raise _bad(op, "the last dimension must be 1 .. 16384")
    if x.numel() // x.shape[-1] > _ROWS_MAX:
        raise _bad(op, "more than 2^31 - 1 rows")
    if tuple(weight.shape) != (x.shape[-1],):
        raise _bad(op, f"weight {tuple(weight.shape)} does not match input {tuple(x.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise _bad(op, f"residual {tuple(residual.shape)} and input {tuple(x.shape)} differ (it is not broadcast)")
    _same_place(op, x, residual, weight)
    half = _half_type(op, x, residual, weight, out)
    if x.dtype == torch.float32 and residual is not None and residual.dtype != torch.float32:
        raise _bad(op, "a float32 input needs a float32 residual")
    if out is not None and out != x.dtype and x.dtype != torch.float32:
        raise _bad(op, f"out_dtype {out} of a {x.dtype} input")
    return half


def _rms_norm_forward(x, residual, weight, eps, out_dtype):
    half = _norm_check("rms_norm", x, residual, weight, out_dtype)
    x2 = _rows(x)
    y = torch.empty(x.shape, device=x.device, dtype=out_dtype or x.dtype)
    rstd = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    h = torch.empty(x.shape if residual is not None else 0, device=x.device, dtype=x.dtype if residual is None else residual.dtype)
    _launch(ops.rmsnorm_fwd, x.device, half, x2, None if residual is None else _rows(residual), weight.contiguous(),
            None if residual is None else h, y, rstd, float(eps))
    return y, h, rstd


def _rms_norm_forward_fake(x, residual, weight, eps, out_dtype):
    _norm_check("rms_norm", x, residual, weight, out_dtype)
    return (x.new_empty(x.shape, dtype=out_dtype or x.dtype), x.new_empty(0) if residual is None else residual.new_empty(residual.shape),
            x.new_empty(x.shape[:-1], dtype=torch.float32))


def _rms_norm_backward(dy, dh, h, weight, rstd, x_dtype, need_x, need_residual, need_weight):
    """(dx, dresidual, dweight), empty where not wanted; where x and the stream have one type the two gradients are one tensor, dx."""
    D = h.shape[-1]
    h2, dy2 = h.reshape(-1, D).contiguous(), dy.reshape(-1, D).contiguous()
    dh2 = None if dh is None else dh.to(h.dtype).reshape(-1, D).contiguous()
    # the kernel's dx has dy's type; a 16-bit output of an f32 x has its gradient from f32 dy, so that dx is f32
    if dy2.dtype != x_dtype:
        dy2 = dy2.to(x_dtype)
    one = x_dtype == h.dtype
    dx = torch.empty(h.shape, device=h.device, dtype=x_dtype) if need_x or (one and need_residual) else None
    dres = torch.empty(h.shape, device=h.device, dtype=h.dtype) if need_residual and not one else None
    dw = torch.empty(D, device=h.device, dtype=weight.dtype) if need_weight else None
    w = weight.contiguous()
    half = _half_type("rms_norm", dy2, h2, w)
    _launch(ops.rmsnorm_bwd, h.device, half, dy2, dh2, h2, w, rstd, dx, dres, dw)
    none = torch.empty(0, device=h.device)
    return tuple(none if t is None else t for t in (dx, dres, dw)) if dx is not None or dres is not None or dw is not None else (none, none, none)


def _rms_norm_backward_fake(dy, dh, h, weight, rstd, x_dtype, need_x, need_residual, need_weight):
    one = x_dtype == h.dtype
    return (h.new_empty(h.shape if need_x or (one and need_residual) else 0, dtype=x_dtype),
            h.new_empty(h.shape if need_residual and not one else 0), weight.new_empty(weight.shape if need_weight else 0))


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, out_dtype):
        y, h, rstd = torch.ops.mvit.rms_norm_forward.default(x, residual, weight, eps, out_dtype)
        ctx.save_for_backward(x if residual is None else h, weight, rstd)
        ctx.x_dtype, ctx.residual = x.dtype, residual is not None
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(rstd)
        if residual is None:
            ctx.mark_non_differentiable(h)
        return y, h, rstd

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh, _):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_res, need_w = ctx.needs_input_grad[:3]
        if dy is None:      # y was not used: the stream's gradient alone
            if dh is None:
                return None, None, None, None, None
            return (dh.to(ctx.x_dtype) if need_x else None, dh if need_res else None, torch.zeros_like(weight) if need_w else None, None, None)
        dx, dres, dw = torch.ops.mvit.rms_norm_backward.default(dy, dh, h, weight, rstd, ctx.x_dtype, need_x, need_res, need_w)
        if need_res and ctx.x_dtype == h.dtype:
            dres = dx
        return dx if need_x else None, dres if need_res else None, dw if need_w else None, None, None


_define("rms_norm_backward(Tensor dy, Tensor? dh, Tensor h, Tensor weight, Tensor rstd, ScalarType x_dtype, bool need_x, bool need_residual, "
        "bool need_weight) -> (Tensor, Tensor, Tensor)", _rms_norm_backward, _rms_norm_backward_fake)
_RMS_NORM = _define("rms_norm_forward(Tensor x, Tensor? residual, Tensor weight, float eps, ScalarType? out_dtype) -> (Tensor, Tensor, Tensor)",
                    _rms_norm_forward, _rms_norm_forward_fake, _RmsNorm)


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension (1 .. 16384), statistics in f32.

    x: bf16, fp16 or f32; weight: f32 or the 16-bit type.  The output has x's type; an f32 x (a residual stream) may ask for a 16-bit
    output with out_dtype.  Differentiable in x and weight."""
    return _RMS_NORM(x, None, weight, eps, out_dtype)[0]


def add_rms_norm(x: Tensor, residual: Tensor, weight: Tensor, eps: float = 1e-6,
                 out_dtype: Optional[torch.dtype] = None) -> tuple[Tensor, Tensor]:
    """(y, h): h = x + residual in the residual's type, y = rms_norm(h) in x's type -- a branch's output joins the residual stream and the
    stream is normed for the next branch, in one pass.  What is normed is h as it is stored.

    x: bf16, fp16 or f32; residual: x's shape, x's type or f32.  Differentiable in x, residual and weight, through y and h."""
    y, h, _ = _RMS_NORM(x, residual, weight, eps, out_dtype)
    return y, h


def _rms_norm_fp8(x, residual, weight, eps):
    _no_grad("rms_norm_fp8", x, residual, weight)
    half = _norm_check("rms_norm_fp8", x, residual, weight)
    q = torch.empty(x.shape, device=x.device, dtype=_E4M3)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    h = torch.empty(x.shape if residual is not None else 0, device=x.device, dtype=x.dtype if residual is None else residual.dtype)
    _launch(ops.rmsnorm_fp8_fwd, x.device, half, _rows(x), None if residual is None else _rows(residual), weight.contiguous(),
            None if residual is None else h, q, scale, float(eps))
    return q, scale, h


def _rms_norm_fp8_fake(x, residual, weight, eps):
    _norm_check("rms_norm_fp8", x, residual, weight)
    return (x.new_empty(x.shape, dtype=_E4M3), x.new_empty(x.shape[:-1], dtype=torch.float32),
            x.new_empty(0) if residual is None else residual.new_empty(residual.shape))


_RMS_NORM_FP8 = _define("rms_norm_fp8(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)", _rms_norm_fp8,
                        _rms_norm_fp8_fake)


def rms_norm_fp8(x: Tensor, weight: Tensor, eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """(q, scale): rms_norm(x) as e4m3 values with one f32 scale a row, y = q * scale[..., None]; what ``linear_fp8`` takes.

    scale = max(max |y|, 1e-30) / 448, q = y / scale rounded to nearest even.  A row with a NaN or an infinity reads back as NaN.
    Serving only (no gradient)."""
    q, scale, _ = _RMS_NORM_FP8(x, None, weight, eps)
    return q, scale


def add_rms_norm_fp8(x: Tensor, residual: Tensor, weight: Tensor, eps: float = 1e-6) -> tuple[Tensor, Tensor, Tensor]:
    """(q, scale, h): ``add_rms_norm`` with its output in 8 bits as ``rms_norm_fp8`` gives it.  Serving only (no gradient)."""
    return _RMS_NORM_FP8(x, residual, weight, eps)


def _quantize_check(op, x):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 16384:
        raise _bad(op, "the last dimension must be 1 .. 16384")
    if x.numel() // x.shape[-1] > _ROWS_MAX:
        raise _bad(op, "more than 2^31 - 1 rows")
    return _half_type(op, x)


def _quantize_fp8(x):
    _no_grad("quantize_fp8", x)
    half = _quantize_check("quantize_fp8", x)
    q = torch.empty(x.shape, device=x.device, dtype=_E4M3)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    _launch(ops.quantize_rows_fp8, x.device, half, _rows(x), q, scale)
    return q, scale


def _quantize_fp8_fake(x):
    _quantize_check("quantize_fp8", x)
    return x.new_empty(x.shape, dtype=_E4M3), x.new_empty(x.shape[:-1], dtype=torch.float32)


_QUANTIZE_FP8 = _define("quantize_fp8(Tensor x) -> (Tensor, Tensor)", _quantize_fp8, _quantize_fp8_fake)


def quantize_fp8(x: Tensor) -> tuple[Tensor, Tensor]:
    """(q, scale): the rows of x (bf16, fp16 or f32; last dimension 1 .. 16384) as e4m3 values with one f32 scale each, as
    ``rms_norm_fp8`` gives them: activations that no norm precedes, and the weights of ``linear_fp8``.  Serving only (no gradient)."""
    return _QUANTIZE_FP8(x)


# ------------------------------------------------------------------ rotary positions
def _rotary_check(op, x, positions, inv_freq, sections, rotate_heads, num_prefix):
    if x.dim() != 4:
        raise _bad(op, f"x must be [B, N, heads, head_dim], got {tuple(x.shape)}")
    B, N, H, Dh = x.shape
    if Dh % 2 or not 2 <= Dh <= 1024 or not 1 <= H <= 1024 or B > 65535 or N > _ROWS_MAX:
        raise _bad(op, "head_dim must be even and at most 1024, heads 1 .. 1024, batch at most 65535")
    pairs = sum(sections)
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or not 1 <= pairs <= Dh // 2:
        raise _bad(op, f"sections {list(sections)}: 1 to 4 axes, together 1 .. head_dim / 2 pairs")
    if not 0 <= rotate_heads <= H or not 0 <= num_prefix <= N:
        raise _bad(op, f"rotate_heads {rotate_heads} of {H}, num_prefix {num_prefix} of {N}")
    want = (N - num_prefix, len(sections))
    if tuple(positions.shape) not in (want, (B, *want)):
        raise _bad(op, f"positions must be {list(want)} or {[B, *want]}, got {list(positions.shape)}")
    if positions.dtype not in ops._POS_TYPES:
        raise _bad(op, f"positions are int32, int64 or float32, got {positions.dtype}")
    if tuple(inv_freq.shape) != (pairs,) or inv_freq.dtype not in (torch.float32, torch.float64):
        raise _bad(op, f"inv_freq must be float32 or float64 [{pairs}], got {inv_freq.dtype} {list(inv_freq.shape)}")
    _same_place(op, x, positions, inv_freq)
    return _half_type(op, x)


def _rotary_into(half, x, y, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse):
    if x.numel():
        _launch(ops.rotary, x.device, half, x, y, positions.contiguous(), inv_freq.contiguous(), sections, rotate_heads, num_prefix, interleaved,
                inverse)
    return y


def _rotary(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse):
    half = _rotary_check("rotary", x, positions, inv_freq, sections, rotate_heads, num_prefix)
    if x.stride(3) != 1:
        x = x.contiguous()
    return _rotary_into(half, x, torch.empty_like(x), positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse)


def _rotary_fake(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse):
    _rotary_check("rotary", x, positions, inv_freq, sections, rotate_heads, num_prefix)
    return torch.empty_like(x if x.stride(3) == 1 else x.contiguous())


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.rest = (sections, rotate_heads, num_prefix, interleaved, not inverse)
        return torch.ops.mvit.rotary_forward.default(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse)

    @staticmethod
    def backward(ctx, dy):   # the turn is linear and orthogonal: its gradient is the turn back (differentiable again by itself)
        return (torch.ops.mvit.rotary_forward.default(dy, *ctx.saved_tensors, *ctx.rest), *(None,) * 7)


_ROTARY = _define("rotary_forward(Tensor x, Tensor positions, Tensor inv_freq, int[] sections, int rotate_heads, int num_prefix, bool interleaved, "
                  "bool inverse) -> Tensor", _rotary, _rotary_fake, _Rotary)


def rotary(x: Tensor, positions: Tensor, inv_freq: Tensor, sections: Sequence[int], rotate_heads: Optional[int] = None, num_prefix: int = 0,
           interleaved: bool = False) -> Tensor:
    """Rotary positions with 1 to 4 axes on x [B, N, heads, head_dim] (any strides; bf16, fp16 or f32).

    Pair i of a head -- values (i, i + P), or (2i, 2i + 1) where interleaved, P = sum(sections) <= head_dim / 2 -- turns by
    positions[token, axis of i] * inv_freq[i]; sections[a] consecutive pairs belong to axis a, values from 2P on pass through.
    positions: [N - num_prefix, axes] or [B, N - num_prefix, axes], int32, int64 or float32; inv_freq: [P], float64 or float32
    (``rotary_frequencies``).  The first num_prefix tokens (class, registers) and the heads from rotate_heads on (default: none) pass
    through, so that attention's packed projection is turned in one call:

        qkv = rotary(qkv.view(B, N, 3 * H, Dh), positions, inv_freq, sections, 2 * H, num_prefix).view(B, N, -1)

    Angles are formed and reduced in f64, so that far positions keep theirs.  Differentiable in x."""
    return _ROTARY(x, positions, inv_freq, sections, x.shape[2] if rotate_heads is None and x.dim() == 4 else rotate_heads or 0, num_prefix,
                   interleaved, False)


def _rotary_inplace(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved):
    _no_grad("rotary_", x)
    half = _rotary_check("rotary_", x, positions, inv_freq, sections, rotate_heads, num_prefix)
    if x.stride(3) != 1 or any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape)):
        raise _bad("rotary_", "x must have dense heads and no expanded dimension to be turned in place")
    _rotary_into(half, x, x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, False)
    return x


def _rotary_inplace_fake(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved):
    _rotary_check("rotary_", x, positions, inv_freq, sections, rotate_heads, num_prefix)
    return x


_ROTARY_ = _define("rotary_(Tensor(a!) x, Tensor positions, Tensor inv_freq, int[] sections, int rotate_heads, int num_prefix, bool interleaved) "
                   "-> Tensor(a!)", _rotary_inplace, _rotary_inplace_fake)


def rotary_(x: Tensor, positions: Tensor, inv_freq: Tensor, sections: Sequence[int], rotate_heads: Optional[int] = None, num_prefix: int = 0,
            interleaved: bool = False) -> Tensor:
    """``rotary`` in place, for serving (no gradient): what passes through is neither read nor written."""
    return _ROTARY_(x, positions, inv_freq, sections, x.shape[2] if rotate_heads is None and x.dim() == 4 else rotate_heads or 0, num_prefix,
                    interleaved)


def rotary_frequencies(sections: Sequence[int], base: float = 10000.0, shared: bool = False, device=None) -> Tensor:
    """inv_freq of ``rotary``: each axis has a spectrum of its own, base^(-j / sections[a]) for its pairs j (the axes of an image), or all
    pairs share one that the sections cut up, base^(-i / P) for pair i (time, height and width of a video)."""
    if shared:
        n = sum(sections)
        exps = [i / n for i in range(n)]
    else:
        exps = [j / n for n in sections for j in range(n)]
    return torch.tensor([float(base) ** -e for e in exps], dtype=torch.float64, device=device)


def grid_positions(*sizes: int, device=None) -> Tensor:
    """int32 positions [prod(sizes), len(sizes)] of a grid in row-major order: (rows, columns) of patches, (time, height, width)."""
    axes = torch.meshgrid(*(torch.arange(n, dtype=torch.int32, device=device) for n in sizes), indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes], -1)


# ------------------------------------------------------------------ linear with activation and residual
def _linear_check(op, x, weight, bias, residual, activation, multiple):
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[1] % multiple or not weight.numel():
        raise _bad(op, f"weight {tuple(weight.shape)} does not match input {tuple(x.shape)} (K must be a multiple of {multiple})")
    K, N = weight.shape[1], weight.shape[0]
    if K * weight.element_size() > 2 ** 23 or N > _ROWS_MAX or x.numel() // K > _ROWS_MAX:
        raise _bad(op, "K is at most 2^23 bytes, N and the rows of x at most 2^31 - 1")
    if activation not in ops.ACTIVATIONS:
        raise _bad(op, f"activation {activation!r}: one of {sorted(ops.ACTIVATIONS)}")
    if bias is not None and tuple(bias.shape) != (N,):
        raise _bad(op, f"bias {tuple(bias.shape)}, expected {(N,)}")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], N):
        raise _bad(op, f"residual {tuple(residual.shape)}, expected {(*x.shape[:-1], N)} (it is not broadcast)")
    _same_place(op, x, weight, bias, residual)


def _operand(t):
    """[rows, K] view for the matrix kernels: rows that start on 16 bytes and are at most 2^23 bytes apart, a copy where they do not"""
    t = _rows(t)
    es = t.element_size()
    if t.data_ptr() % 16 or (t.shape[0] > 1 and (t.stride(0) * es % 16 or t.stride(0) * es > 2 ** 23)):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _linear_half(op, x, weight, bias, residual):
    if x.dtype not in _HALF or weight.dtype != x.dtype:
        raise _bad(op, f"x and weight are both bfloat16 or both float16, got {x.dtype} and {weight.dtype}")
    return _half_type(op, x, bias, residual)


def _linear_act_forward(x, weight, bias, residual, activation, save_pre):
    op = "linear_act"
    _linear_check(op, x, weight, bias, residual, activation, 8)
    half = _linear_half(op, x, weight, bias, residual)
    y = torch.empty((*x.shape[:-1], weight.shape[0]), device=x.device, dtype=x.dtype if residual is None else residual.dtype)
    pre = torch.empty(y.shape if save_pre else 0, device=x.device, dtype=x.dtype)
    if y.numel():
        _launch(ops.linear_act, x.device, half, _operand(x), _operand(weight), None if bias is None else bias.contiguous(),
                None if residual is None else _rows(residual), y, pre if save_pre else None, activation)
    return y, pre


def _linear_act_forward_fake(x, weight, bias, residual, activation, save_pre):
    _linear_check("linear_act", x, weight, bias, residual, activation, 8)
    _linear_half("linear_act", x, weight, bias, residual)
    y = x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=x.dtype if residual is None else residual.dtype)
    return y, x.new_empty(y.shape if save_pre else 0)


def _linear_products(dz, x, weight, need_x, need_w):
    """dx = dz @ weight and dweight = dz^T @ x"""
    (M, N), K = dz.shape, weight.shape[1]
    dx = dw = None
    if need_x:
        ld = -(-N // 8) * 8      # the K axis of this product: padded to whole pieces, the padding times zeros
        wt = torch.empty(K, ld, device=dz.device, dtype=dz.dtype) if ld == N else torch.zeros(K, ld, device=dz.device, dtype=dz.dtype)
        ops.transpose_bf16(weight, wt, N, K, weight.stride(0), ld)
        if ld != N:
            dz_p = torch.zeros(M, ld, device=dz.device, dtype=dz.dtype)
            dz_p[:, :N] = dz
        else:
            dz_p = dz
        dx = torch.empty(M, K, device=dz.device, dtype=dz.dtype)
        ops.linear_act(dz_p, wt, None, None, dx, None, "none")
    if need_w:
        ld = -(-M // 8) * 8
        dzt, xt = (torch.zeros(n, ld, device=dz.device, dtype=dz.dtype) if ld != M else torch.empty(n, ld, device=dz.device, dtype=dz.dtype)
                   for n in (N, K))
        ops.transpose_bf16(dz, dzt, M, N, dz.stride(0), ld)
        ops.transpose_bf16(x, xt, M, K, x.stride(0), ld)
        dw = torch.empty(N, K, device=dz.device, dtype=dz.dtype)
        ops.linear_act(dzt, xt, None, None, dw, None, "none")
    return dx, dw


def _linear_act_backward(dy, x, weight, pre, activation, need_x, need_w, need_b, bias_dtype):
    N, K = weight.shape
    dev, dt = x.device, x.dtype
    dx = torch.empty(x.shape if need_x else 0, device=dev, dtype=dt)
    dw = torch.empty((N, K) if need_w else 0, device=dev, dtype=dt)
    db = torch.empty(N if need_b else 0, device=dev, dtype=bias_dtype)
    dy2 = dy.reshape(-1, N).contiguous()
    M = dy2.shape[0]
    if M == 0:
        return dx, dw.zero_(), db.zero_()
    z = None if activation == "none" else pre.reshape(-1, N)
    products = need_x or need_w
    dz = dy2
    if z is not None or dy2.dtype != dt or need_b:
        dz = torch.empty(M, N, device=dev, dtype=dt) if products and (z is not None or dy2.dtype != dt) else None
        _launch(ops.act_bwd, dev, dt, dy2, z, activation, dz, db if need_b else None)
        dz = dy2 if dz is None else dz
    if products:
        got = _launch(_linear_products, dev, dt, dz, _operand(x), _operand(weight), need_x, need_w)
        dx = got[0].view(x.shape) if need_x else dx
        dw = got[1] if need_w else dw
    return dx, dw, db


def _linear_act_backward_fake(dy, x, weight, pre, activation, need_x, need_w, need_b, bias_dtype):
    return (x.new_empty(x.shape if need_x else 0), weight.new_empty(weight.shape if need_w else 0),
            x.new_empty(weight.shape[0] if need_b else 0, dtype=bias_dtype))


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, save_pre):
        keep = activation != "none" and any(ctx.needs_input_grad[:3])
        y, pre = torch.ops.mvit.linear_act_forward.default(x, weight, bias, residual, activation, keep)
        ctx.save_for_backward(x, weight, pre)
        ctx.activation, ctx.bias_dtype = activation, None if bias is None else bias.dtype
        ctx.mark_non_differentiable(pre)
        return y, pre

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _):
        x, weight, pre = ctx.saved_tensors
        need_x, need_w, need_b, need_res = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            dx, dw, db = torch.ops.mvit.linear_act_backward.default(dy, x, weight, pre, ctx.activation, need_x, need_w, need_b,
                                                                    ctx.bias_dtype or x.dtype)
        return dx if need_x else None, dw if need_w else None, db if need_b else None, dy if need_res else None, None, None


_define("linear_act_backward(Tensor dy, Tensor x, Tensor weight, Tensor pre, str activation, bool need_x, bool need_w, bool need_b, "
        "ScalarType bias_dtype) -> (Tensor, Tensor, Tensor)", _linear_act_backward, _linear_act_backward_fake)
_LINEAR_ACT = _define("linear_act_forward(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str activation, bool save_pre) -> (Tensor, Tensor)",
                      _linear_act_forward, _linear_act_forward_fake, _LinearAct)


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None, activation: str = "none") -> Tensor:
    """residual + act(x @ weight^T + bias) in one launch; act: none, relu, silu, gelu (erf) or gelu_tanh.

    x [..., K], weight [N, K]: both bf16 or both fp16, K a multiple of 8; bias [N] and residual [..., N]: that type or f32.  The output has
    the residual's type (f32: a residual stream), else x's.  f32 accumulation, one rounding at the end.  Differentiable in x, weight, bias
    and residual; the value in front of the activation is kept in 16 bits for it."""
    return _LINEAR_ACT(x, weight, bias, residual, activation, False)[0]


def _linear_fp8_check(x, x_scale, weight, w_scale, bias, residual, activation, out_dtype):
    op = "linear_fp8"
    if x.dtype != _E4M3 or weight.dtype != _E4M3:
        raise _bad(op, f"x and weight are float8_e4m3fn, got {x.dtype} and {weight.dtype}")
    _linear_check(op, x, weight, bias, residual, activation, 16)
    if x_scale.dtype != torch.float32 or w_scale.dtype != torch.float32 or x_scale.shape != x.shape[:-1] or w_scale.shape != weight.shape[:1]:
        raise _bad(op, f"float32 scales {tuple(x.shape[:-1])} and {tuple(weight.shape[:1])}, got {x_scale.dtype} {tuple(x_scale.shape)} and "
                       f"{w_scale.dtype} {tuple(w_scale.shape)}")
    _same_place(op, x, x_scale, w_scale)
    if out_dtype not in (*_HALF, torch.float32):
        raise _bad(op, f"out_dtype {out_dtype}")
    return _half_type(op, bias, residual, *(() if residual is not None else (out_dtype,)))


def _linear_fp8(x, x_scale, weight, w_scale, bias, residual, activation, out_dtype):
    _no_grad("linear_fp8", x_scale, w_scale, bias, residual)
    half = _linear_fp8_check(x, x_scale, weight, w_scale, bias, residual, activation, out_dtype)
    y = torch.empty((*x.shape[:-1], weight.shape[0]), device=x.device, dtype=out_dtype if residual is None else residual.dtype)
    if y.numel():
        _launch(ops.linear_act, x.device, half, _operand(x), _operand(weight), None if bias is None else bias.contiguous(),
                None if residual is None else _rows(residual), y, None, activation, x_scale.contiguous(), w_scale.contiguous())
    return y


def _linear_fp8_fake(x, x_scale, weight, w_scale, bias, residual, activation, out_dtype):
    _linear_fp8_check(x, x_scale, weight, w_scale, bias, residual, activation, out_dtype)
    return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=out_dtype if residual is None else residual.dtype)


_LINEAR_FP8 = _define("linear_fp8(Tensor x, Tensor x_scale, Tensor weight, Tensor w_scale, Tensor? bias, Tensor? residual, str activation, "
                      "ScalarType out_dtype) -> Tensor", _linear_fp8, _linear_fp8_fake)


def linear_fp8(x: Tensor, x_scale: Tensor, weight: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None,
               activation: str = "none", out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``linear_act`` with e4m3 operands: residual + act((x @ weight^T) * x_scale[..., None] * w_scale + bias).

    x [..., K] with x_scale [...] and weight [N, K] with w_scale [N], as ``quantize_fp8``, ``rms_norm_fp8`` and ``add_rms_norm_fp8`` give
    them; K a multiple of 16.  The output has the residual's type, else out_dtype (bf16, fp16 or f32).  Serving only (no gradient)."""
    return _LINEAR_FP8(x, x_scale, weight, w_scale, bias, residual, activation, out_dtype)


__all__ = ["rms_norm", "add_rms_norm", "rms_norm_fp8", "add_rms_norm_fp8", "quantize_fp8", "rotary", "rotary_", "rotary_frequencies",
           "grid_positions", "linear_act", "linear_fp8"]
