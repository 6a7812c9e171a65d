"""The experts of a mixture-of-experts layer on MXFP4 rows: products grouped by expert with
a fused epilogue, their gradients, and the weighted way back to token order.

No reference counterpart: the reference converts the permuted MXFP4 rows to FP8 and hands
them to Transformer Engine's grouped GEMM.  Outputs are allocated on the call and filled by
the sm_100a kernels through `omo`, on torch's current stream, without host synchronisation:
`m_splits` (rows per expert, in the order of the rows) stays on the device.
"""
from __future__ import annotations

from typing import Optional

import torch

import mxfp4_b200  # noqa: F401
from mxfp4_b200.capi import ACTIVATIONS
from omo import omo_bias_act_grad_new as _act_grad_op
from omo import omo_grouped_gemm_mxfp4_new as _gemm_op
from omo import omo_grouped_wgrad_mxfp4 as _wgrad_op
from omo import omo_moe_unpermute_grad_new as _unpermute_grad_op
from omo import omo_moe_unpermute_new as _unpermute_op
from omo import omo_swizzle_scales_grouped as _swizzle_op

uint8_type = torch.uint8


def _activation(name: str) -> int:
    if name not in ACTIVATIONS:
        raise RuntimeError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]


def omo_swizzle_scales_grouped(scales: torch.Tensor, gated: bool = False) -> torch.Tensor:
    """E8M0 scales of stacked weights [E, N, K/32], as the rowwise quantizer writes them, in
    the 128x4-tile layout that `omo_grouped_gemm_mxfp4` reads; `gated` weights (gate rows
    above up rows, activation "swiglu") have each half in tiles of its own.  Once per
    weight update."""
    E, N, S = scales.shape
    parts = 2 if gated else 1
    out = torch.empty((E, parts * ((N // parts + 127) // 128 * 128), (S + 3) // 4 * 4),
                      device=scales.device, dtype=uint8_type)
    _swizzle_op(scales.contiguous(), parts, out)
    return out


def omo_grouped_gemm_mxfp4(a_codes: torch.Tensor, a_scales: torch.Tensor, b_codes: torch.Tensor,
                           b_scales: torch.Tensor, m_splits: Optional[torch.Tensor],
                           bias: Optional[torch.Tensor] = None, activation: str = "none",
                           residual: Optional[torch.Tensor] = None, save_pre: bool = False,
                           quantize: bool = False, bf16_out: bool = True):
    """act(A . B_e^T + bias_e) + residual for the rows of every expert e.

    a_codes [M, K/2] and a_scales [M, K/32]: rows sorted by expert, as the quantizer or
    `omo_moe_permute_mxfp4` returns them (rows may be strided); m_splits int32 [E] on the
    device; b_codes [E, N, K/2] with b_scales from `omo_swizzle_scales_grouped`; bias [E, N]
    BF16 or FP32; residual BF16 [M, W], W = N, or N/2 with "swiglu".  Activations: none,
    relu, relu2, silu, gelu, gelu_tanh, swiglu.

    Returns the BF16 result [M, W], followed where asked for by the BF16 rows before the
    activation [M, N] (`save_pre`) and the result's rowwise MXFP4, codes [M, W/2] and scales
    [M, W/32] (`quantize`); `bf16_out=False` leaves the BF16 result out.  Rows past the sum
    of m_splits are not written."""
    out = _gemm_op(a_codes, a_scales, m_splits, b_codes, b_scales, bias, _activation(activation),
                   residual, save_pre, quantize, bf16_out)
    return out[0] if len(out) == 1 else tuple(out)


def omo_gemm_mxfp4_act(a_codes: torch.Tensor, a_scales: torch.Tensor, b_codes: torch.Tensor,
                       b_scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       activation: str = "none", residual: Optional[torch.Tensor] = None,
                       save_pre: bool = False, quantize: bool = False, bf16_out: bool = True):
    """One dense layer: act(A . B^T + bias) + residual with b_codes [N, K/2], b_scales [its
    128x4-tile rows, ...] and bias [N]; otherwise as `omo_grouped_gemm_mxfp4`.  Any number of
    rows, N % 8 == 0 (swiglu: N % 16 == 0), K % 32 == 0."""
    return omo_grouped_gemm_mxfp4(a_codes, a_scales, b_codes, b_scales, None, bias, activation,
                                  residual, save_pre, quantize, bf16_out)


def omo_grouped_wgrad_mxfp4(dy: torch.Tensor, x_codes: torch.Tensor, x_scales: torch.Tensor,
                            m_splits: Optional[torch.Tensor],
                            out_dtype: torch.dtype = torch.float32,
                            accumulate_into: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dw[e] = dy_e^T . x_e over the rows of every expert e: dy BF16 [M, N], x the MXFP4 rows
    saved by the forward pass.  Returns dw [E, N, K] in FP32 or BF16; `accumulate_into` (FP32
    [E, N, K]) is added to and returned instead.  m_splits None: one group of all rows."""
    if accumulate_into is not None:
        _wgrad_op(dy, x_codes, x_scales, m_splits, accumulate_into, True)
        return accumulate_into
    E = 1 if m_splits is None else m_splits.shape[0]
    dw = torch.empty((E, dy.shape[1], x_codes.shape[1] * 2), device=dy.device, dtype=out_dtype)
    _wgrad_op(dy, x_codes, x_scales, m_splits, dw, False)
    return dw


def omo_bias_act_grad(dy: torch.Tensor, pre: Optional[torch.Tensor],
                      m_splits: Optional[torch.Tensor], activation: str = "none",
                      bias_grad: bool = True, quantize: bool = False, bf16_out: bool = True):
    """The gradient of the epilogue: dz = dy * act'(pre) and, with `bias_grad`, dbias [E, N]
    FP32 = the sum of dz over every expert's rows.  Returns (dz, dbias, codes, scales) without
    what was not asked for; codes [M, N/2] and scales [M, N/32] (`quantize`) are the rowwise
    MXFP4 of dz, the left operand of the input gradient's product."""
    out = _act_grad_op(dy, pre, m_splits, _activation(activation), bias_grad, quantize, bf16_out)
    return out[0] if len(out) == 1 else tuple(out)


def omo_moe_unpermute(y: torch.Tensor, row_map: torch.Tensor,
                      weight: Optional[torch.Tensor] = None,
                      topk: Optional[int] = None) -> torch.Tensor:
    """out[t] = sum over k of weight[t, k] * y[row_map[t, k]], the way back of
    `omo_moe_permute_mxfp4` with its `dst` (negative or too large: no row).  y BF16 [R, H],
    row_map int32 [T, topk], weight FP32 [T, topk] or None (ones); `topk` takes the first
    columns of a wider map (a row_id_map: topk = E)."""
    return _unpermute_op(y, row_map, weight, row_map.shape[1] if topk is None else topk)


def omo_moe_unpermute_grad(dout: torch.Tensor, y: torch.Tensor, row_map: torch.Tensor,
                           weight: Optional[torch.Tensor] = None, topk: Optional[int] = None,
                           weight_grad: bool = True, quantize: bool = False,
                           zero_unnamed: bool = False):
    """The gradient of `omo_moe_unpermute`: dy[row_map[t, k]] = weight[t, k] * dout[t] and, with
    `weight_grad`, dweight [T, topk] FP32 = <dout[t], y[row_map[t, k]]> (0 without a row).
    Returns (dy, dweight, codes, scales) without what was not asked for; codes and scales
    (`quantize`) are dy's rowwise MXFP4.  Rows that row_map does not name are left
    uninitialised, or zero with `zero_unnamed`."""
    out = _unpermute_grad_op(dout, y, row_map, weight, row_map.shape[1] if topk is None else topk,
                             weight_grad, quantize, zero_unnamed)
    return out[0] if len(out) == 1 else tuple(out)
