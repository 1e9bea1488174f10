"""The 8-bit activation path: int8 activations (one scale a row) in front of
the int8 weights of ``Int8Linear``.

The W8A16 GEMM multiplies 16-bit activations.  With the activations in 8 bits
too, a long prompt's products run on the int8 tensor cores and move half the
activation bytes.  The path of a decoder layer's MLP:

* ``add_rmsnorm_int8`` -- the residual's addition, the RMSNorm and the
  quantization of every row, in one pass (``add_rmsnorm``: the same with a
  16-bit output, in front of the W8A16 GEMM or ``int8_moe``);
* ``int8_gemm_w8a8`` -- gate and up;
* ``swiglu_int8`` -- ``silu(gate) * up`` and its quantization, in one pass;
* ``int8_gemm_w8a8`` -- down.

``Int8SwiGLU.forward_w8a8`` runs the last three.  rotalabs-accel quantizes
weights only (src/rotalabs_accel/kernels/gemm.py:189-238); its pieces that
these join are ``rmsnorm`` (kernels/normalization.py:186-213), ``swiglu_fused``
(kernels/activations.py:109-137) and ``quantize_symmetric``
(quantization/symmetric.py:24-82), whose convention the int8 rows follow:
``scale = max|v| / 127``, a zero row gets scale 1, round half to even.

CUDA tensors run the sm_100a kernels (fp16 or bf16 activations); CPU tensors
the same formulas in torch operations (fp32 activations too, which the kernels
refuse: a residual stream would lose bits in a cast).  For inference: no
gradients flow, on either.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _capi


def _quantize_rows(v: torch.Tensor):
    """fp32 rows -> (int8 rows, fp32 scale of each); a row with an infinity or
    NaN gets the scale NaN and zeros."""
    if v.shape[-1] == 0:
        return v.to(torch.int8), torch.ones(v.shape[:-1], dtype=torch.float32, device=v.device)
    scale = v.abs().amax(dim=-1) / 127
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    scale = torch.where(torch.isfinite(scale), scale, torch.full_like(scale, float("nan")))
    q = torch.round(v / scale.unsqueeze(-1)).clamp(-127, 127)
    return torch.nan_to_num(q, nan=0.0).to(torch.int8), scale


def _silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up``, rounded once to fp32 (``silu`` of a gate below -88
    is beyond fp32's range; times a large ``up`` it may not be)."""
    return (torch.nn.functional.silu(gate.double()) * up.double()).float()


def _rows(x: Optional[torch.Tensor]):
    """``(..., K)`` as ``(rows, K)`` (None stays None)."""
    return None if x is None else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def _norm_torch(x, residual, weight, eps):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    return hf * torch.rsqrt(hf.pow(2).mean(dim=-1, keepdim=True) + eps) * weight.float(), h


def _norm_args(x, residual, weight):
    assert x.shape[-1] == weight.shape[0], f"Hidden dim mismatch: {x.shape[-1]} vs {weight.shape[0]}"
    assert residual is None or residual.shape == x.shape, \
        f"Residual shape mismatch: {tuple(residual.shape)} vs {tuple(x.shape)}"


def _swiglu_args(gate, up):
    assert gate.shape == up.shape, f"Gate and up shape mismatch: {tuple(gate.shape)} vs {tuple(up.shape)}"


def _w8a8_args(x_int8, x_scale, weight_int8, scale):
    assert x_int8.dtype == torch.int8, "Activations must be INT8"
    assert weight_int8.dtype == torch.int8, "Weight must be INT8"
    K, N = x_int8.shape[-1], weight_int8.shape[0]
    assert weight_int8.shape == (N, K), f"Weight shape mismatch: {weight_int8.shape} vs ({N}, {K})"
    assert x_scale.shape == x_int8.shape[:-1], \
        f"Activation scale shape mismatch: {tuple(x_scale.shape)} vs {tuple(x_int8.shape[:-1])}"
    assert scale.shape == (N,), f"Scale shape mismatch: {scale.shape} vs ({N},)"


# 2-D CUDA operands, the per-token case, go straight to the extension, which
# checks them; what it refuses is checked once more here, so that a mismatch of
# shapes is the same AssertionError everywhere.

def add_rmsnorm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6):
    """``h = x + residual`` (rounded to ``x.dtype``; ``x`` itself where
    ``residual`` is None) and ``y = rmsnorm(h)``: returns ``(y, h)``, both of
    ``x.dtype``.

    x, residual: ``(..., K)`` fp16 or bf16 (the same); weight ``(K,)`` fp32,
    fp16 or bf16.  The norm is taken of the rounded sum, in fp32."""
    if x.is_cuda and x.dim() == 2:
        try:
            return _capi.torch_ops().add_rmsnorm(x, residual, weight, eps)
        except RuntimeError:
            _norm_args(x, residual, weight)
            raise
    _norm_args(x, residual, weight)
    if x.is_cuda:
        y, h = _capi.torch_ops().add_rmsnorm(_rows(x), _rows(residual), weight, eps)
        return y.view(x.shape), x if residual is None else h.view(x.shape)
    with torch.no_grad():
        v, h = _norm_torch(x, residual, weight, eps)
        return v.to(x.dtype), h


def add_rmsnorm_int8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6):
    """``add_rmsnorm`` with the normalized rows in int8: returns ``(q, scale,
    h)`` with ``q`` int8 ``(..., K)``, ``scale`` fp32 ``(...)`` (one a row,
    ``max|row| / 127``, 1 for a zero row) and ``h`` as in ``add_rmsnorm``.
    ``q * scale`` is what ``int8_gemm_w8a8`` multiplies.  A row holding an
    infinity or NaN gets the scale NaN and ``q = 0``."""
    if x.is_cuda and x.dim() == 2:
        try:
            return _capi.torch_ops().add_rmsnorm_int8(x, residual, weight, eps)
        except RuntimeError:
            _norm_args(x, residual, weight)
            raise
    _norm_args(x, residual, weight)
    if x.is_cuda:
        q, s, h = _capi.torch_ops().add_rmsnorm_int8(_rows(x), _rows(residual), weight, eps)
        return q.view(x.shape), s.view(x.shape[:-1]), x if residual is None else h.view(x.shape)
    with torch.no_grad():
        v, h = _norm_torch(x, residual, weight, eps)
        q, s = _quantize_rows(v)
        return q, s, h


def swiglu_int8(gate: torch.Tensor, up: torch.Tensor):
    """``silu(gate) * up`` (fp32) in int8: returns ``(q, scale)`` as
    ``add_rmsnorm_int8`` does.  gate, up: ``(..., N)`` fp16 or bf16."""
    if gate.is_cuda and gate.dim() == 2:
        try:
            return _capi.torch_ops().swiglu_int8(gate, up)
        except RuntimeError:
            _swiglu_args(gate, up)
            raise
    _swiglu_args(gate, up)
    if gate.is_cuda:
        q, s = _capi.torch_ops().swiglu_int8(_rows(gate), _rows(up))
        return q.view(gate.shape), s.view(gate.shape[:-1])
    with torch.no_grad():
        return _quantize_rows(_silu_mul(gate, up))


def int8_gemm_w8a8(x_int8: torch.Tensor, x_scale: torch.Tensor, weight_int8: torch.Tensor, scale: torch.Tensor,
                   bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """W8A8 GEMM ``y = (x_int8 * x_scale) @ (weight_int8 * scale).T + bias``.

    x_int8: int8 ``(..., K)``; x_scale: fp32 ``(...)``, one a row;
    weight_int8: int8 ``(N, K)``; scale: ``(N,)`` fp32 or fp16; bias: optional
    ``(N,)`` fp16 or fp32.  Returns fp16 ``(..., N)``.  The sum over K is
    exact (int32), so K < 131072; any strides, sizes and alignment (rows that
    are not 16-byte aligned are copied first)."""
    if x_int8.is_cuda and x_int8.dim() == 2:
        try:
            return _capi.torch_ops().w8a8_gemm(x_int8, x_scale, weight_int8, scale, bias)
        except RuntimeError:
            _w8a8_args(x_int8, x_scale, weight_int8, scale)
            raise
    _w8a8_args(x_int8, x_scale, weight_int8, scale)
    if x_int8.is_cuda:
        y = _capi.torch_ops().w8a8_gemm(_rows(x_int8), x_scale.reshape(x_scale.numel()), weight_int8, scale, bias)
        return y.view(*x_int8.shape[:-1], weight_int8.shape[0])
    with torch.no_grad():
        # products of int8 summed in fp64: exact, as on the GPU
        y = (x_int8.double() @ weight_int8.double().t()).float() * scale.float() * x_scale.unsqueeze(-1)
        return (y if bias is None else y + bias.float()).half()
