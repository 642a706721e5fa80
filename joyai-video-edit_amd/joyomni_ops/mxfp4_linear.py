"""MXFP4 linear layer on the gfx950 kernels: ``Fp8Linear``'s counterpart with 4-bit weights and
activations (microscaled E2M1, one power-of-two scale for 32 elements along K).

* weights are quantised once, [N, K] row by row, and kept as the (K / 2, N) column-major view of their codes;
* activations are quantised per call, or arrive quantised from the operator before
  (``fused_norm_scale_shift_mxfp4``, ``gemm_quant``);
* ``y = round(sum + bias)`` in fp32 up to the one rounding, with the epilogues of the block: GELU-tanh,
  GELU-tanh quantised for the next layer, gated residual.

Codes and scales are laid out as ``per_block_quant_mxfp4`` describes; ``scales_from_row_major`` takes those of a
checkpoint that keeps one scale per [row, block].
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import (mxfp4_scaled_mm, mxfp4_scaled_mm_gated_residual, mxfp4_scaled_mm_gelu_tanh,
               mxfp4_scaled_mm_gelu_tanh_quant, per_block_quant_mxfp4)

CODE_DTYPE = torch.float4_e2m1fn_x2
SCALE_DTYPE = torch.float8_e8m0fnu
BLOCK = 32  # elements of a scale
SLAB = 256  # elements of a row in one slab of scales


def empty_mxfp4(rows: int, K: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes [rows, K / 2] and scales [ceil(K / 256), rows, 8] to be written by an operator."""
    if K % BLOCK:
        raise ValueError(f"K must be a multiple of {BLOCK}, the MXFP4 block, not {K}")
    return (torch.empty(rows, K // 2, dtype=CODE_DTYPE, device=device),
            torch.empty(-(-K // SLAB), rows, SLAB // BLOCK, dtype=SCALE_DTYPE, device=device))


def quantize_mxfp4(x_2d: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] bf16 / fp16 / fp32 on the GPU -> (codes, scales)."""
    q, s = empty_mxfp4(x_2d.shape[0], x_2d.shape[1], x_2d.device)
    per_block_quant_mxfp4(x_2d, q, s)
    return q, s


def scales_from_row_major(scales: torch.Tensor) -> torch.Tensor:
    """E8M0 scales [rows, K / 32] -> the operators' [ceil(K / 256), rows, 8], unused bytes 0."""
    if scales.dim() != 2 or scales.element_size() != 1:
        raise ValueError("scales must be [rows, K / 32] of one byte each")
    rows, blocks = scales.shape
    per = SLAB // BLOCK
    out = torch.zeros(-(-blocks // per) * per, rows, dtype=torch.uint8, device=scales.device)
    out[:blocks] = scales.view(torch.uint8).t()
    return out.view(-1, per, rows).permute(0, 2, 1).contiguous().view(SCALE_DTYPE)


def scales_to_row_major(scales: torch.Tensor, K: int) -> torch.Tensor:
    """The operators' scales of K elements a row -> [rows, K / 32]."""
    s = scales.view(torch.uint8).permute(1, 0, 2).reshape(scales.shape[1], -1)
    return s[:, : K // BLOCK].contiguous().view(SCALE_DTYPE)


class MxFp4Linear(nn.Module):
    def __init__(self, weight_q: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor],
                 out_dtype: torch.dtype = torch.bfloat16, gelu_tanh: bool = False):
        """weight_q (K / 2, N) column-major codes, weight_scale [ceil(K / 256), N, 8], bias [N] of out_dtype."""
        super().__init__()
        self.register_buffer("weight_q", weight_q, persistent=False)
        self.register_buffer("weight_scale", weight_scale, persistent=False)
        if bias is not None:
            self.register_buffer("bias", bias.contiguous(), persistent=False)
        else:
            self.bias = None
        self.out_dtype = out_dtype
        self.gelu_tanh = gelu_tanh
        self.in_features = weight_q.shape[0] * 2
        self.out_features = weight_q.shape[1]

    @classmethod
    def from_linear(cls, lin: nn.Linear, out_dtype: torch.dtype = torch.bfloat16,
                    gelu_tanh: bool = False) -> "MxFp4Linear":
        q, s = quantize_mxfp4(lin.weight.data)
        b = lin.bias.data.to(dtype=out_dtype) if lin.bias is not None else None
        return cls(q.t(), s, b, out_dtype=out_dtype, gelu_tanh=gelu_tanh)

    def gemm(self, x_q: torch.Tensor, x_scale: torch.Tensor) -> torch.Tensor:
        """The product (+ fused epilogue) on quantised activations."""
        mm = mxfp4_scaled_mm_gelu_tanh if self.gelu_tanh else mxfp4_scaled_mm
        return mm(x_q, self.weight_q, x_scale, self.weight_scale, self.out_dtype, self.bias)

    def gemm_quant(self, x_q: torch.Tensor, x_scale: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """GELU-tanh of the product, quantised in its epilogue: the next layer's (x_q, x_scale)."""
        assert self.gelu_tanh, "only the GELU epilogue is quantised in place"
        q, s = empty_mxfp4(x_q.shape[0], self.out_features, x_q.device)
        mxfp4_scaled_mm_gelu_tanh_quant(x_q, self.weight_q, x_scale, self.weight_scale, self.bias, q, s)
        return q, s

    def gemm_gated_residual(self, x_q: torch.Tensor, x_scale: torch.Tensor, residual: torch.Tensor,
                            gate: torch.Tensor, inplace: bool = False) -> torch.Tensor:
        """residual + gemm(x_q, x_scale) * gate in the product's epilogue; residual [M, N], in place contiguous
        and 16-byte aligned."""
        assert not self.gelu_tanh, "the gated-residual epilogue has no GELU"
        assert residual.dtype == self.out_dtype, "residual dtype must be the output dtype"
        return mxfp4_scaled_mm_gated_residual(x_q, self.weight_q, x_scale, self.weight_scale, residual, gate,
                                              self.bias, inplace)

    def _quantize(self, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        x_2d = x.reshape(-1, x.shape[-1])
        assert x_2d.shape[1] == self.in_features, f"in features mismatch {x_2d.shape[1]} vs {self.in_features}"
        rows_apart = x_2d.stride(1) == 1 and x_2d.stride(0) >= self.in_features
        return quantize_mxfp4(x_2d if rows_apart else x_2d.contiguous())

    def gated_residual(self, x: torch.Tensor, residual: torch.Tensor, gate: torch.Tensor,
                       inplace: bool = False) -> torch.Tensor:
        """residual + self(x) * gate: x [M, K] quantised, then one product."""
        return self.gemm_gated_residual(*self._quantize(x), residual, gate, inplace)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.gemm(*self._quantize(x)).reshape(*x.shape[:-1], self.out_features)
