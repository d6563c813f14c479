"""Normalization layers for the rocm backend on the HIP kernels.

LayerNorm      -- the nn.LayerNorm signature and state dict (``weight``, ``bias``), normalizing
                  the last dimension (difflet/backends/cpu/ops_impl/norm.py:9); fp32 statistics.
RMSNorm        -- (hidden_size, eps=1e-6) with one ``weight`` (the state dict of
                  difflet/backends/cpu/ops_impl/norm.py:12-22); computed with the fp32 law of
                  the CUDA backend (difflet/backends/cuda/ops_impl/norm.py:28-44): fp32
                  statistics, normalisation and affine, one cast back. The CPU module
                  normalises in the input dtype; the two agree within bf16 rounding.
rms_norm_fp32  -- difflet/backends/_torch_megatron/norm.py:35-45 on the kernel.
rms_norm_quantized -- RMSNorm of a residual sum, written as the 8-bit operand of an fp8 linear.
"""

from __future__ import annotations

import numbers

import torch
import torch.nn as nn

from difflet_amd.backends.rocm.ops_impl import library


def rms_norm_fp32(x: torch.Tensor, weight: torch.Tensor | None, eps: float) -> torch.Tensor:
    if x.shape[-1] % 8:
        raise NotImplementedError(f"rocm rms_norm needs the last dim a multiple of 8, got {x.shape[-1]}")
    return library.rms_norm(x, weight, float(eps))


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor | None, eps: float, *,
                       residual: torch.Tensor | None = None, format: str = "fp8_rowwise"
                       ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """RMSNorm of ``x + residual`` over the last dim in one pass: (codes, scales, hidden).

    codes (float8_e4m3fn, x's shape) and scales are the activation operand of an fp8 linear:
    ``format="fp8_rowwise"`` fp32 scales, one per row; ``"mxfp8"`` uint8 E8M0 scales, one per block
    of 32, codes and blocks in the swizzle order of the quantized weights. The norm is rounded once,
    to e4m3. hidden is ``x + residual`` in x's dtype, the next residual stream (x without one).
    x bf16, fp16 or fp32, residual like it; the last dim a multiple of 8 (mxfp8: 128) up to 16384."""
    if format not in ("fp8_rowwise", "mxfp8"):
        raise ValueError(f"format must be 'fp8_rowwise' or 'mxfp8', got {format!r}")
    mx = format == "mxfp8"
    if x.device.type != "cuda":
        raise ValueError(f"rocm rms_norm takes device tensors, got one on {x.device}")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise NotImplementedError(f"rocm rms_norm runs bf16 / fp16 / fp32; got {x.dtype}")
    dim = x.shape[-1] if x.dim() else 0
    if dim == 0 or dim % (128 if mx else 8) or dim > 16384:
        raise NotImplementedError(f"rocm rms_norm to {format} needs the last dim a multiple of "
                                  f"{128 if mx else 8} up to 16384, got {dim}")
    if weight is not None and (weight.dim() != 1 or weight.shape[0] != dim):
        raise ValueError(f"weight must be [{dim}], got {tuple(weight.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must be {x.dtype} {tuple(x.shape)}, got {residual.dtype} "
                         f"{tuple(residual.shape)}")
    if x.dim() == 2:
        q, s, h = library.rms_norm_quant(x, weight, residual, float(eps), mx)
        return q, s, x if residual is None else h
    r2 = None if residual is None else residual.reshape(-1, dim)
    q, s, h = library.rms_norm_quant(x.reshape(-1, dim), weight, r2, float(eps), mx)
    lead = x.shape[:-1]
    return (q.reshape(x.shape), s.reshape(*lead, dim // 32) if mx else s.reshape(lead),
            x if residual is None else h.reshape(x.shape))


class RMSNorm(nn.Module):
    def __init__(self, hidden_size: int, eps: float = 1e-6, **kwargs):
        super().__init__()
        del kwargs
        self.weight = nn.Parameter(torch.ones(hidden_size))
        self.eps = eps

    def forward(self, hidden_states: torch.Tensor) -> torch.Tensor:
        return rms_norm_fp32(hidden_states, self.weight, self.eps)


CustomRMSNorm = RMSNorm


class LayerNorm(nn.Module):
    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, device=None, dtype=None):
        super().__init__()
        if isinstance(normalized_shape, numbers.Integral):
            normalized_shape = (int(normalized_shape),)
        self.normalized_shape = tuple(normalized_shape)
        if len(self.normalized_shape) != 1:
            raise NotImplementedError("rocm LayerNorm normalizes the last dimension only")
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        factory = {"device": device, "dtype": dtype}
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(self.normalized_shape, **factory))
            self.bias = nn.Parameter(torch.zeros(self.normalized_shape, **factory)) if bias else None
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"LayerNorm over {self.normalized_shape}, got input {tuple(x.shape)}")
        if x.shape[-1] % 8:
            raise NotImplementedError("rocm LayerNorm needs the last dim a multiple of 8")
        return library.layer_norm(x, self.weight, self.bias, float(self.eps))

    def extra_repr(self) -> str:
        return f"{self.normalized_shape}, eps={self.eps}, elementwise_affine={self.elementwise_affine}"


__all__ = ["CustomRMSNorm", "LayerNorm", "RMSNorm", "rms_norm_fp32", "rms_norm_quantized"]
