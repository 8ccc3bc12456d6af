"""Dropout whose mask is a function of a seed and an offset: it is formed again where it is needed and never stored."""
import torch
from torch import Tensor

__all__ = ["dropout"]

K = torch.ops.mamtorch_kernel_encoder


def word(v: int) -> int:
    """A number modulo 2^64, as the operators' signed 64-bit argument."""
    v = int(v) & 0xFFFFFFFFFFFFFFFF
    return v - (1 << 64) if v >> 63 else v


def default_scale(p: float) -> float:
    """1 / (1 - p); 0 where nothing is kept."""
    return 1.0 / (1.0 - p) if p < 1 else 0.0


def dropout(x: Tensor, p: float, seed: int, offset: int = 0, residual: Tensor = None, scale: float = None, step: Tensor = None) -> Tensor:
    """``x`` with elements dropped with probability ``p`` (rounded to a multiple of 2^-32) and the others times ``scale`` (default
    1 / (1 - p)), plus ``residual`` where one is given.

    Element i of the contiguous order of x's shape takes word i % 4 of Philox4x32-10 with counter (i / 4, offset) and key ``seed``, so equal
    arguments give equal masks on any tensor of that size; a training loop takes another ``offset`` for each call.  ``step``: one int64
    element on the GPU that is added to the offset when the kernel runs: under a HIP graph, whose replays repeat
    the arguments, advance it between replays."""
    return K.dropout.default(x, residual, float(p), default_scale(p) if scale is None else float(scale), word(seed), word(offset), step)


@torch.library.register_fake("mamtorch_kernel_encoder::dropout")
def _(x, residual, p, scale, seed, offset, step):
    torch._check(residual is None or (residual.shape == x.shape and residual.dtype == x.dtype))
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)
