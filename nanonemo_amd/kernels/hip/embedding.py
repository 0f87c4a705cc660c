"""The model's embedding on the gfx950 kernels (include/nanonemo_embedding.h): the lookup with a scale, and its gradient by
sorted tokens.

``embedding(idx, weight, scale, padding_idx)`` stands for ``F.embedding(idx, weight, padding_idx) * scale``
(/root/reference/nanonemo/model/model.py:13-70 has it without a scale): the product in fp32, rounded once. Its gradient is
summed in fp32 and rounded once, whatever the weight's type, in an order that the tokens and sizes alone decide:
bit-reproducible, where PyTorch adds 16-bit rows in 16 bits or with atomics. The model selects it with ``emb_kernel="hip"``.

A token that is not in [0, V) makes its row of the output NaN and takes no part in the gradient (F.embedding ends the
process with a device assertion). Tokens are int64 or int32. Once differentiable, in reverse mode: a tangent is refused.
Capturing a call that autograd records into a HIP graph is refused, as the attention's is; without autograd it captures.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import forward_ad

from nanonemo_amd.kernels.hip import eager, host, preload, refuse_capture, refuse_forward_ad


@torch.library.custom_op("nanonemo::embedding", mutates_args=())
def _embedding(idx: Tensor, weight: Tensor, scale: float, padding_idx: int) -> Tensor:
    return host().embedding_fwd(idx, weight, scale)


@_embedding.register_fake
def _(idx, weight, scale, padding_idx):
    return weight.new_empty((*idx.shape, weight.shape[1]))


@torch.library.custom_op("nanonemo::embedding_bwd", mutates_args=())
def _embedding_bwd(d_out: Tensor, idx: Tensor, rows: int, scale: float, padding_idx: int) -> Tensor:
    return host().embedding_bwd(d_out, idx, rows, scale, padding_idx)


@_embedding_bwd.register_fake
def _(d_out, idx, rows, scale, padding_idx):
    return d_out.new_empty((rows, d_out.shape[-1]))


def _save(ctx, idx, weight, scale, padding_idx):
    ctx.save_for_backward(idx)
    ctx.call = (weight.shape[0], scale, padding_idx)


def _setup_context(ctx, inputs, output):
    refuse_capture("embedding (autograd)")
    _save(ctx, *inputs)


def _backward(ctx, d_out):
    refuse_capture("embedding backward")
    return None, _embedding_bwd(d_out, *ctx.saved_tensors, *ctx.call), None, None


_embedding.register_autograd(_backward, setup_context=_setup_context)


def embedding(idx: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: int | None = None) -> Tensor:
    """scale * weight[idx]: idx (...) int64 or int32, weight (V, N) fp16, bf16 or fp32 -> (..., N) of the weight's type.
    Rows whose token is ``padding_idx`` (negative: from the end) give the weight no gradient."""
    rows = weight.shape[0]
    if padding_idx is None:
        padding_idx = -1
    elif -rows <= padding_idx < rows:
        padding_idx %= rows
    else:
        raise ValueError(f"padding_idx {padding_idx} is not a row of the weight ({rows} rows)")
    if forward_ad._current_level >= 0:
        refuse_forward_ad("embedding", weight)
    if eager(idx, weight):  # the same launches as the op's, as one autograd node of the host module
        return host().embedding(idx, weight, scale, padding_idx)
    refuse_capture("embedding", weight)
    return _embedding(idx, weight, scale, padding_idx)


preload()
