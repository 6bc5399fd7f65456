"""Operators of a transformer block beside ``linear``, ``layer_norm`` and ``attention`` of ``torch_ops``: the RMS norm of a residual
stream (with an 8-bit output for serving), 8-bit quantisation of rows, rotary positions with several axes, and the linear layer with
activation and residual in its epilogue, in 16 and in 8 bits.

They are ``torch.ops.mvit.*`` operators like those, with shape (meta) implementations and autograd formulas on the backward kernels; the
functions below are their entry points, re-exported by ``torch_ops``.  CUDA (ROCm) tensors only.  16-bit operands are bf16 or fp16 as
the tensors are (fp16 runs in libmiphei_hip_f16.so), never a mixture; the work goes to the tensors' device, on its current stream.  Wrong
arguments raise ValueError.

Their gradients are those of a backward pass, once.  Forward-mode tangents and functional gradient transforms (torch.func.grad, vjp, jvp) are
refused by all of them, not dropped; torch.vmap runs those without a gradient an entry at a time.

All of them can be captured into a graph, forward and backward; as with any backward pass, let no eager graph over the same leaves live
while one is captured (delete its outputs first): its accumulation nodes belong to the eager stream.

Checks, allocations, autograd formulas and the calls of the C-ABI are in csrc/torch_ops.cpp (libmiphei_torch.so), not in Python: a call on
one token costs its host time.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional, Sequence

import torch
from torch import Tensor

from . import _lib as L

TORCH_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libmiphei_torch.so")


class _Missing:
    def __init__(self, why):
        self.why = why

    def __call__(self, *args):
        raise RuntimeError(self.why)


def _load():
    """Registers the operators and binds them to the two libraries; where a library is missing, every call says so (no fallback)."""
    build = "build it with `python -c 'import __graft_entry__ as g; g.build()'` (hipcc --offload-arch=gfx950). The MI355X path has no fallback."
    for path in (TORCH_LIB_PATH, L.LIB_PATH, L.LIB_PATH_F16):
        if not os.path.exists(path):
            return f"{path} is missing: {build}"
    torch.ops.load_library(TORCH_LIB_PATH)
    bind = ctypes.CDLL(TORCH_LIB_PATH).mvit_torch_bind
    bind.argtypes, bind.restype = [ctypes.c_char_p, ctypes.c_char_p], ctypes.c_char_p
    why = bind(os.fsencode(L.LIB_PATH), os.fsencode(L.LIB_PATH_F16))
    return None if why is None else f"{why.decode()}: {build}"


_WHY = _load()


def _op(name):
    return getattr(torch.ops.mvit, name).default if _WHY is None else _Missing(_WHY)


_RMS_NORM, _RMS_NORM_FP8, _QUANTIZE_FP8 = _op("rms_norm_forward"), _op("rms_norm_fp8"), _op("quantize_fp8")
_ROTARY, _ROTARY_, _LINEAR_ACT, _LINEAR_FP8 = _op("rotary_forward"), _op("rotary_"), _op("linear_act_forward"), _op("linear_fp8")


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


def rms_norm_fp8(x: Tensor, weight: Tensor, eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """(q, scale): rms_norm(x) as e4m3 values with one f32 scale a row, y = q * scale[..., None]; what ``linear_fp8`` takes.

    scale = max(max |y|, 1e-30) / 448, q = y / scale rounded to nearest even.  A row with a NaN or an infinity reads back as NaN.
    Serving only (no gradient)."""
    q, scale, _ = _RMS_NORM_FP8(x, None, weight, eps)
    return q, scale


def add_rms_norm_fp8(x: Tensor, residual: Tensor, weight: Tensor, eps: float = 1e-6) -> tuple[Tensor, Tensor, Tensor]:
    """(q, scale, h): ``add_rms_norm`` with its output in 8 bits as ``rms_norm_fp8`` gives it.  Serving only (no gradient)."""
    return _RMS_NORM_FP8(x, residual, weight, eps)


def quantize_fp8(x: Tensor) -> tuple[Tensor, Tensor]:
    """(q, scale): the rows of x (bf16, fp16 or f32; last dimension 1 .. 16384) as e4m3 values with one f32 scale each, as
    ``rms_norm_fp8`` gives them: activations that no norm precedes, and the weights of ``linear_fp8``.  Serving only (no gradient)."""
    return _QUANTIZE_FP8(x)


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


def rotary_(x: Tensor, positions: Tensor, inv_freq: Tensor, sections: Sequence[int], rotate_heads: Optional[int] = None, num_prefix: int = 0,
            interleaved: bool = False) -> Tensor:
    """``rotary`` in place, for serving (no gradient): what passes through is neither read nor written."""
    _ROTARY_(x, positions, inv_freq, sections, x.shape[2] if rotate_heads is None and x.dim() == 4 else rotate_heads or 0, num_prefix, interleaved)
    return x


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


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None, activation: str = "none") -> Tensor:
    """residual + act(x @ weight^T + bias) without intermediate results in memory (but where a long K is taken in parts); act: none, relu,
    silu, gelu (erf) or gelu_tanh.

    x [..., K], weight [N, K]: both bf16 or both fp16, K a multiple of 8 (at most 2^22, and so N; at most 2^29 rows of x where weight's
    gradient is wanted); bias [N] and residual [..., N]: that type or f32.  The output has
    the residual's type (f32: a residual stream), else x's.  f32 accumulation, one rounding at the end.  Differentiable in x, weight, bias
    and residual: the value in front of the activation is kept in 16 bits for it whatever the output's type, and its gradient is rounded to 16 bits in
    front of the products for x and weight (not of bias' sum).

    ``torch_ops.linear`` beside it rounds what it is given (f32 masters too) to bf16 and gives dweight in the weight's type, summed in f32; where x
    and weight are 16-bit tensors already this is the faster of the two (forward and backward of [5264, 1536] x [4096, 1536] 202 us, that 538) and
    keeps fp16 as it is."""
    return _LINEAR_ACT(x, weight, bias, residual, activation, False)[0]


def linear_fp8(x: Tensor, x_scale: Tensor, weight: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None,
               activation: str = "none", out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``linear_act`` with e4m3 operands: residual + act((x @ weight^T) * x_scale[..., None] * w_scale + bias).

    x [..., K] with x_scale [...] and weight [N, K] with w_scale [N], as ``quantize_fp8``, ``rms_norm_fp8`` and ``add_rms_norm_fp8`` give
    them; K a multiple of 16.  The output has the residual's type, else out_dtype (bf16, fp16 or f32).  An f32 output is formed on the 16-bit matrix
    instructions, exactly but for f32 sums; a 16-bit one may be formed on the e4m3 instructions, by its size: they keep 13 bits below the largest of
    neighbouring products, less than the output's rounding shows of the products' magnitudes.  Serving only (no gradient)."""
    return _LINEAR_FP8(x, x_scale, weight, w_scale, bias, residual, activation, out_dtype)


__all__ = ["rms_norm", "add_rms_norm", "rms_norm_fp8", "add_rms_norm_fp8", "quantize_fp8", "rotary", "rotary_", "rotary_frequencies",
           "grid_positions", "linear_act", "linear_fp8"]
