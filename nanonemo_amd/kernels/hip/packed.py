"""Causal GQA attention over packed sequences on the gfx950 kernels (include/nanonemo_packed.h).

Documents or prompts of different lengths lie one behind the other in (tokens, heads, hd) tensors, without padding, and every
token attends to its own sequence up to itself. The reference's model has batches of one length only
(/root/reference/nanonemo/kernels/cuda/flash_attn.py:18-60).

    packing = Packing([417, 1024, 3], heads=12, kv_heads=4)      # once per batch
    o = flash_attn_packed(q, k, v, packing)                        # q (1444, 12, hd), k, v (1444, 4, hd)

A ``Packing`` holds how the kernels share the work out, on the host and on the device: tiles and units of the longest
sequences first, long ones split where they would outlast the others. The kernels are the dense attention's, so a sequence's
output is the same bits as flash_attn's on it alone, and everything is deterministic. The gradients are nearer to the formula's
than the dense ones: the forward keeps what rounding its output to 16 bits took off, one byte a value, for rowsum(dO * o) (where
a wave has a sequence's whole rows in the backward, up to 32 tokens, it keeps nothing: those bytes are left as they were).

fp16 or bf16, head_dim 32 or 64, sequences of 0 to 2^30 / (H hd) tokens. Once differentiable, in reverse mode (a tangent is
refused); capturing a call that autograd records into a HIP graph is refused, as the dense attention's is; without autograd it
captures, with the packing that it was given.
"""

from __future__ import annotations

import operator

import torch
from torch import Tensor
from torch.autograd import forward_ad

from nanonemo_amd.kernels.hip import eager, host, preload, records, refuse_capture, refuse_forward_ad

_POSITIONS = 15  # the word of a plan that says where the positions begin (NN_FA_PACKED_POSITIONS)


class Packing:
    """How sequences of the given lengths (>= 0) lie in a packed batch, for attention with these heads on this device. Its
    tensors are not to be changed. They are copied on the device's current stream and, as any tensor's are, their memory is that
    stream's: another stream waits for it before it uses them, and they are kept until it has, and as long as a captured graph.

    lengths    the lengths, a tuple;   tokens   their sum;   longest   the longest
    positions  (tokens,) int32 on the device: each token's position in its sequence
    """

    def __init__(self, lengths, heads: int, kv_heads: int, device: torch.device | str = "cuda"):
        self.lengths = tuple(operator.index(n) for n in (lengths.tolist() if isinstance(lengths, Tensor) else lengths))
        self.tokens, self.longest = sum(self.lengths), max(self.lengths, default=0)
        self.heads, self.kv_heads = heads, kv_heads
        device = torch.device(device)
        if device.type == "cuda" and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("Packing: made while a HIP graph is captured, whose replays would copy it again from memory that is gone; make it before")
        with torch.inference_mode(False):  # (autograd saves the plan, which it does with no inference tensor)
            self.plan_host = host().packed_plan(self.lengths, heads, kv_heads)
            # (from pinned memory, which its allocator keeps until the copy has run: the host does not wait)
            self.plan = self.plan_host.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else self.plan_host
            self.positions = self.plan[int(self.plan_host[_POSITIONS]) :]

    @property
    def device(self) -> torch.device:
        return self.plan.device

    def __repr__(self) -> str:
        return f"Packing({len(self.lengths)} sequences, {self.tokens} tokens, heads={self.heads}, kv_heads={self.kv_heads}, device={self.device})"


@torch.library.custom_op("nanonemo::flash_attn_packed", mutates_args=())
def _flash_attn_packed(q: Tensor, k: Tensor, v: Tensor, plan: Tensor, plan_host: Tensor, backward: bool) -> tuple[Tensor, Tensor, Tensor]:
    return host().packed_fwd(q, k, v, plan, plan_host, backward)


@_flash_attn_packed.register_fake
def _(q, k, v, plan, plan_host, backward):
    T, H, _ = q.shape
    return (
        torch.empty(q.shape, dtype=q.dtype, device=q.device),
        torch.empty((H, T), dtype=torch.float32, device=q.device),
        torch.empty(q.shape if backward else 0, dtype=torch.int8, device=q.device),
    )


@torch.library.custom_op("nanonemo::flash_attn_packed_bwd", mutates_args=())
def _flash_attn_packed_bwd(
    d_o: Tensor, q: Tensor, k: Tensor, v: Tensor, o: Tensor, lse: Tensor, rest: Tensor, plan: Tensor, plan_host: Tensor
) -> tuple[Tensor, Tensor, Tensor]:
    return host().packed_bwd(d_o, q, k, v, o, lse, rest, plan, plan_host)


@_flash_attn_packed_bwd.register_fake
def _(d_o, q, k, v, o, lse, rest, plan, plan_host):
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))


def _setup_context(ctx, inputs, output):
    refuse_capture("flash_attn_packed (autograd)")
    q, k, v, plan, plan_host, _ = inputs
    ctx.save_for_backward(q, k, v, *output, plan, plan_host)
    ctx.set_materialize_grads(False)  # lse's gradient is ignored


def _backward(ctx, d_o, _d_lse, _d_rest=None):
    refuse_capture("flash_attn_packed backward")
    if d_o is None:
        return (None,) * 6
    return *_flash_attn_packed_bwd(d_o, *ctx.saved_tensors), None, None, None


_flash_attn_packed.register_autograd(_backward, setup_context=_setup_context)


def flash_attn_packed(q: Tensor, k: Tensor, v: Tensor, packing: Packing) -> Tensor:
    """Causal GQA attention within each of the packing's sequences: q (tokens, H, hd), k and v (tokens, KVH, hd), fp16 or bf16,
    -> (tokens, H, hd), contiguous. Column ranges of a projection are read in place where q is one, or k and v both are;
    in the backward q is copied unless the gradient of the output has its strides."""
    if forward_ad._current_level >= 0:
        refuse_forward_ad("flash_attn_packed", q, k, v)
    if eager(q, k, v):  # the same launches as the op's, as one autograd node of the host module
        return host().packed(q, k, v, packing.plan, packing.plan_host)
    refuse_capture("flash_attn_packed", q, k, v)
    return _flash_attn_packed(q, k, v, packing.plan, packing.plan_host, records(q, k, v))[0]


preload()
