"""Dropout without stored masks: a counter-based generator on the device (csrc/philox.cuh).

The reference draws LoRA dropout with ``torch.native_dropout`` on the padded batch and keeps the mask
(solution/varlen.py:42-63, solution/attn.py:130-203), which stays the default here. The Functions
below take a generator state instead, (seed, offset) as an int64 [2] tensor on the device; a mask is
a function of the state, a stream number and the value's index, and the backward pass computes it
again. Nothing is drawn from torch's generators.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops
from ._state import STATE

STREAMS = 1 << 20  # of one packed forward: its dropouts take them one after the other


class CounterRNG:
    """The state of the generator on one device. ``take(n)`` returns the state for the next n streams
    (numbers 0 .. n - 1) as a tensor of its own and advances; both are enqueued on the current stream,
    so a captured step draws new masks at each replay. Ranks of a data-parallel job take different
    seeds."""

    def __init__(self, seed: int | None = None, device="cuda"):
        seed = torch.initial_seed() if seed is None else int(seed)
        seed = (seed + 2 ** 63) % 2 ** 64 - 2 ** 63  # as int64
        with torch.inference_mode(False):  # a state made in an evaluation serves the training after it
            self.state = torch.tensor([seed, 0], dtype=torch.int64, device=device)

    def take(self, n: int = 1) -> torch.Tensor:
        with torch.inference_mode(False):
            now = self.state.clone()
            self.state[1] += n
        return now


class StepStreams:
    """The streams of one packed forward: the generator's state at its start, and the next stream."""

    def __init__(self, rng: torch.Tensor):
        self.rng, self.next = rng, 0

    def streams(self, n: int):
        """(rng, first stream) of the next n streams."""
        first, self.next = self.next, self.next + n
        if self.next > STREAMS:
            raise RuntimeError(f"decik_b200 dropout: more than {STREAMS} dropouts in one forward")
        return self.rng, first


def step_streams(device):
    """The StepStreams of a packed forward on ``device``, or None while counter-based dropout is off."""
    if STATE.counter_dropout is None:
        return None
    rng = STATE.counter_rngs.get(device)
    if rng is None:
        seed = None if STATE.counter_dropout is True else STATE.counter_dropout
        rng = STATE.counter_rngs[device] = CounterRNG(seed, device)
    return StepStreams(rng.take(STREAMS))


def use_counter_dropout(on=True) -> None:
    """Switch the packed path's dropout to the counter-based generator: ``True`` (seeded by
    torch.initial_seed()) or a seed; False switches back to torch's draws. Dropout on the packed
    decoder (nn.Dropout with 0 < p < 1 and not in place, and the LoRA branches of the attention: in the
    fused block, which then takes layers with LoRA dropout too, in LoRADownDropout for the layers and
    ranks that the block is not for, in their nn.Dropout for what that is not for) draws at the real
    tokens only, stores no mask, and does not touch torch's generators. Each packed forward takes new
    streams. Ranks of a data-parallel job give different seeds."""
    STATE.counter_dropout = None if on is False or on is None else on
    STATE.counter_rngs = {}


class CounterDropout(torch.autograd.Function):
    """dropout(x), or residual + dropout(x), with the mask of (rng, stream): ops.dropout. ``rng`` is kept
    for the backward pass and must not be advanced in place before it (CounterRNG.take's are not)."""

    @staticmethod
    def forward(ctx, x, p, rng, stream=0, residual=None):
        ctx.save_for_backward(rng)
        ctx.meta = (p, stream, x.dtype, residual is not None)
        return ops.dropout(x, p, rng, stream, residual=residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (rng,) = ctx.saved_tensors
        p, stream, dtype, residual = ctx.meta
        return ops.dropout(grad, p, rng, stream, out_dtype=dtype), None, None, None, grad if residual else None


def _rows(t):
    """t [T, W] as the LoRA kernels read it: contiguous rows that start on 16 bytes, one behind the other."""
    if t.dim() != 2:
        return t
    ok = (t.stride(1) == 1 and t.data_ptr() % 16 == 0
          and (t.shape[0] == 1 or (t.stride(0) >= t.shape[1] and t.stride(0) * t.element_size() % 16 == 0)))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


class LoRADownDropout(torch.autograd.Function):
    """The LoRA down projections of x [T, W] under dropout, u [T, branches * rank] =
    scale_b (keep_b x16) A_b^T with a mask for each branch (ops.lora_down_dropout). ``a``: the branches'
    lora_A weights [rank, W] (fp32, as peft keeps them), of one rank, ``p`` the probability of each (a
    number: the same for all), ``dtype`` the compute dtype. Keeps the 16-bit input only."""

    @staticmethod
    def forward(ctx, x, p, rng, stream, dtype, *a):
        p = tuple(p) if isinstance(p, (tuple, list)) else (p,) * len(a)
        if not 1 <= len(a) <= 2 or len(p) != len(a) or any(w.dim() != 2 or w.shape != a[0].shape for w in a):
            raise RuntimeError(f"decik_b200 LoRADownDropout: {len(p)} probabilities for lora_A weights of shapes "
                               f"{[tuple(w.shape) for w in a]} (1 or 2 weights [rank, W] of one rank, a p for each)")
        a16 = torch.cat(a).to(dtype)
        x16, u = ops.lora_down_dropout(_rows(x if x.dtype == dtype else x.float()), a16, p, rng, stream)
        ctx.save_for_backward(x16, a16, rng)
        ctx.meta = (p, stream, x.dtype, [w.dtype for w in a])
        return u

    @staticmethod
    @once_differentiable
    def backward(ctx, du):
        x16, a16, rng = ctx.saved_tensors
        p, stream, x_dtype, a_dtypes = ctx.meta
        dx, da = ops.lora_down_dropout_bwd(_rows(du), x16, a16, p, rng, stream)
        parts = da.split(da.shape[0] // len(a_dtypes))
        return (dx.to(x_dtype), None, None, None, None) + tuple(w.to(t) for w, t in zip(parts, a_dtypes))
