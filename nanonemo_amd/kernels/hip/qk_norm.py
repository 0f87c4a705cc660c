"""Norm of each query and key head with the rotation by position, in one pass, on the gfx950 kernel
(include/nanonemo_qk_norm.h).

``qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)`` stands for RMS norm of every head's vector (in fp32, times
a weight of head_dim values, one for queries and one for keys) followed by the rotation of
/root/reference/nanonemo/model/layers.py:67-74: one rounding, where module by module there are three. The reference's model has
the rotation alone. ``positions`` gives every token's place in its sequence, which in packed batches (kernels/hip/packed.py)
and in steps of decoding is not its index.

A position that is not a row of the tables makes its token's outputs NaN, and its gradients and the weights'. The weights'
gradients are summed in fp32 in an order that the sizes alone decide. Once differentiable, in reverse mode (a tangent is refused);
capturing a call that autograd records into a HIP graph is refused, as the attention's is; without autograd it captures.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from nanonemo_amd.kernels.hip import eager, host, preload, refuse_capture, refuse_forward_ad


def _like(t: Tensor) -> Tensor:
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


@torch.library.custom_op("nanonemo::qk_norm_rope", mutates_args=())
def _qk_norm_rope(
    q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None, eps: float
) -> tuple[Tensor, Tensor]:
    return host().qk_norm_fwd(q, k, q_weight, k_weight, cos, sin, positions, eps)


@_qk_norm_rope.register_fake
def _(q, k, q_weight, k_weight, cos, sin, positions, eps):
    return _like(q), _like(k)


@torch.library.custom_op("nanonemo::qk_norm_rope_bwd", mutates_args=())
def _qk_norm_rope_bwd(
    dq: Tensor, dk: Tensor, q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None, eps: float
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    return host().qk_norm_bwd(dq, dk, q, k, q_weight, k_weight, cos, sin, positions, eps)


@_qk_norm_rope_bwd.register_fake
def _(dq, dk, q, k, q_weight, k_weight, cos, sin, positions, eps):
    return _like(q), _like(k), _like(q_weight), _like(k_weight)


def _setup_context(ctx, inputs, output):
    refuse_capture("qk_norm_rope (autograd)")
    *tensors, ctx.eps = inputs
    ctx.save_for_backward(*tensors)


def _backward(ctx, dq, dk):
    refuse_capture("qk_norm_rope backward")
    return *_qk_norm_rope_bwd(dq, dk, *ctx.saved_tensors, ctx.eps), None, None, None, None


_qk_norm_rope.register_autograd(_backward, setup_context=_setup_context)


def qk_norm_rope(
    q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None = None, eps: float = 1e-5
) -> tuple[Tensor, Tensor]:
    """(rotated norm of q, of k), contiguous: q (T, H, hd) or (B, T, H, hd) and k with KVH heads, fp16, bf16 or fp32, hd a multiple
    of 16 up to 256; weights fp32 (hd,); cos and sin fp32 (T_max, hd/2); positions int64 or int32, (T,) or (B, T), by default
    0 .. T - 1. Column ranges of a projection are read in place."""
    ins = (q, k, q_weight, k_weight, cos, sin)
    if forward_ad._current_level >= 0:
        refuse_forward_ad("qk_norm_rope", *ins)
    if eager(*ins) if positions is None else eager(*ins, positions):  # the op's launches, as one autograd node of the host module
        return host().qk_norm_rope(*ins, positions, eps)
    refuse_capture("qk_norm_rope", *ins[:4])
    return _qk_norm_rope(*ins, positions, eps)


preload()
