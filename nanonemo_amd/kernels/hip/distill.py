"""Distillation from a teacher's top logits on the gfx950 kernels (include/nanonemo_distill.h).

``top_logits(logits, k, temperature)`` is the teacher's side: each row's k largest logits, and the logsumexp of the others at
the temperature. ``distill_loss(logits, values, indices, rest, targets, temperature, weight)`` is the student's: the mean over
the rows of

    weight * temperature^2 * KL(teacher || student) + (1 - weight) * cross entropy of the targets,

read from the student's 16-bit or fp32 logits as they are, once each way, beside ``head_loss``'s cross entropy
(/root/reference/nanonemo/model/model.py:60-66 has the cross entropy alone). Without ``rest`` the teacher's probabilities are
the softmax of its k values; with it, its remaining mass is one class more, compared with the student's mass outside the k.
Without ``targets`` every row counts and the loss is weight * temperature^2 * KL; with them, rows whose target is -100 count
for neither term. Softmax statistics are joined in fp64, since a student near its teacher has a loss far below its logsumexp.

Logits (..., V) may be strided rows (logits[:, :-1]); V up to 393216, k up to 512. An index or target that is out of range
makes the loss and its row's gradient NaN; an index that is there twice adds up its probabilities. The loss is once
differentiable in the logits, in reverse mode (a tangent is refused); the teacher's side takes no gradient. Capturing a call
that autograd records into a HIP graph is refused, as the attention's is; without autograd it captures.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.autograd import forward_ad

from nanonemo_amd.kernels.hip import eager, host, preload, records, refuse_capture, refuse_forward_ad


_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


@torch.library.custom_op("nanonemo::top_logits", mutates_args=())
def _top_logits(logits: Tensor, k: int, temperature: float) -> tuple[Tensor, Tensor, Tensor]:
    return host().top_logits(logits, k, temperature)


@_top_logits.register_fake
def _(logits, k, temperature):
    rows = logits.shape[:-1]
    return logits.new_empty((*rows, k)), logits.new_empty((*rows, k), dtype=torch.int64), logits.new_empty(rows, dtype=torch.float32)


@torch.library.custom_op("nanonemo::distill_loss", mutates_args=())
def _distill_loss(
    logits: Tensor, values: Tensor, indices: Tensor, rest: Tensor | None, targets: Tensor | None, temperature: float, weight: float
) -> tuple[Tensor, Tensor]:
    return host().distill_fwd(logits, values, indices, rest, targets, temperature, weight)


@_distill_loss.register_fake
def _(logits, values, indices, rest, targets, temperature, weight):
    rows = math.prod(logits.shape[:-1])
    return logits.new_empty((), dtype=torch.float32), logits.new_empty(rows * 8 + 1, dtype=torch.float64)


@torch.library.custom_op("nanonemo::distill_loss_bwd", mutates_args=())
def _distill_loss_bwd(
    d_loss: Tensor, logits: Tensor, values: Tensor, indices: Tensor, targets: Tensor | None, stats: Tensor, temperature: float, weight: float
) -> Tensor:
    return host().distill_bwd(d_loss, logits, values, indices, targets, stats, temperature, weight)


@_distill_loss_bwd.register_fake
def _(d_loss, logits, values, indices, targets, stats, temperature, weight):
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


def _save(ctx, inputs, stats):
    logits, values, indices, _, targets, *ctx.call = inputs
    ctx.save_for_backward(logits, values, indices, targets, stats)
    ctx.set_materialize_grads(False)


def _setup_context(ctx, inputs, output):
    refuse_capture("distill_loss (autograd)")
    _save(ctx, inputs, output[1])


def _backward(ctx, d_loss, _d_stats):
    refuse_capture("distill_loss backward")
    none = (None,) * 6
    return (None if d_loss is None else _distill_loss_bwd(d_loss, *ctx.saved_tensors, *ctx.call), *none)


_distill_loss.register_autograd(_backward, setup_context=_setup_context)


def _check_temperature(temperature: float) -> None:
    if not 1e-4 <= temperature <= 1e4:
        raise ValueError(f"temperature must be in [1e-4, 1e4], got {temperature}")


def _check_k(k: int, vocab: int) -> None:
    if not 1 <= k <= min(vocab, 512):
        raise ValueError(f"k must be in [1, min(V, 512)], got {k} of {vocab} logits")


def takes(logits: Tensor, k: int, values: Tensor | None = None, rest: Tensor | None = None) -> bool:
    """Whether logits (..., V) with k of a teacher's are within the kernels' sizes and types; other forms of them exist in
    PyTorch's operations (model.py). What is no valid argument in any form is refused by the functions."""
    V = logits.shape[-1]
    return (logits.dtype in _DTYPES and k <= 512 and V <= 393216 and logits.numel() < V * (1 << 22)
            and (values is None or values.dtype in _DTYPES) and (rest is None or rest.dtype is torch.float32))


def top_logits(logits: Tensor, k: int, temperature: float = 1.0) -> tuple[Tensor, Tensor, Tensor]:
    """(values (..., k) of the logits' type, indices (..., k) int64, rest (...) fp32): the k largest of each row of logits
    (..., V), descending, equal ones by index (NaN above +inf, -0 as 0), and logsumexp(the others / temperature), -inf
    where there are none. Not differentiable: what a frozen teacher gives its student."""
    _check_temperature(temperature)
    _check_k(k, logits.shape[-1])
    logits = logits.detach()
    return host().top_logits(logits, k, temperature) if eager(logits) else _top_logits(logits, k, temperature)


def distill_loss(
    logits: Tensor, values: Tensor, indices: Tensor, rest: Tensor | None = None, targets: Tensor | None = None,
    temperature: float = 1.0, weight: float = 1.0,
) -> Tensor:
    """The distillation loss (see above), an fp32 scalar: logits (..., V) fp16, bf16 or fp32; values and indices (..., k),
    rest (...) as top_logits returns them, at the same temperature; targets (...) int64; weight in [0, 1]."""
    _check_temperature(temperature)
    _check_k(values.shape[-1], logits.shape[-1])
    if not 0.0 <= weight <= 1.0:
        raise ValueError(f"weight must be in [0, 1], got {weight}")
    if weight < 1.0 and targets is None:
        raise ValueError("weight below 1 needs targets, whose cross entropy is the rest of the loss")
    if records(values) or rest is not None and records(rest):
        raise ValueError("the teacher's values take no gradient: detach them")
    if forward_ad._current_level >= 0:
        refuse_forward_ad("distill_loss", logits, values, rest)
    call = (logits, values, indices, rest, targets, float(temperature), float(weight))
    if eager(*(t for t in call[:5] if t is not None)):  # the same launches as the op's, as one autograd node of the host module
        return host().distill(*call)
    refuse_capture("distill_loss", logits)
    return _distill_loss(*call)[0]


preload()
