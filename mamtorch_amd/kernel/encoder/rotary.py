"""Norms of queries and keys for each head, with the position rotation in the same pass."""
import torch
from torch import Tensor

__all__ = ["rotary_frequencies", "norm_rotate"]

K = torch.ops.mamtorch_kernel_encoder


def rotary_frequencies(size: int, base: float = 10000.0, device=None) -> Tensor:
    """``base ** (-2 i / size)`` radians a place for pair i of the ``size`` elements of a head that turn (float64)."""
    if size % 2 or size < 0:
        raise ValueError(f"elements turn in pairs, got {size}")
    return base ** (-torch.arange(0, size, 2, device=device, dtype=torch.float64) / max(size, 1))


def norm_rotate(q: Tensor, k: Tensor, q_weight: Tensor = None, k_weight: Tensor = None, frequencies: Tensor = None, positions: Tensor = None,
                eps: float = 1e-6, norm: bool = True, interleaved: bool = False):
    """Queries and keys with each head normalised by its root mean square, times a weight, and turned by its token's place: for each row of d elements
    ``y = R(place) (x / sqrt(mean(x^2) + eps) * weight)``.

    q (batch, tokens, heads, 2, d), k (batch, tokens, key heads, 2, d), as ``diff_attention`` takes them (each of the two maps is normalised by itself): float32, bfloat16 or
    float16, any strides, d up to 128.  Returns tensors of their shapes.

    q_weight, k_weight (d): of q's type or float32, or None.  norm False: the rotation alone.
    frequencies: float64, radians a place of each pair (``rotary_frequencies``); the first 2 * len(frequencies) elements turn, as pairs (i, i + len) or, interleaved,
    (2 i, 2 i + 1), and the others do not; None: the norm alone.
    positions: int32 (batch, tokens), by default a token's number.  Angles are formed in float64, so that places far out are exact.
    Sums are float32, a result is rounded once, gradients do not depend on the order in which the GPU happens to work.  First derivatives only."""
    return K.norm_rotate.default(q, k, q_weight, k_weight, frequencies, positions, float(eps), bool(norm), bool(interleaved))


TYPES = (torch.float32, torch.bfloat16, torch.float16)


def check_rotation(q, k, q_weight, k_weight, frequencies, positions, norm):
    torch._check(q.dim() == 5 and k.dim() == 5 and q.dtype == k.dtype and q.dtype in TYPES)
    torch._check(k.size(0) == q.size(0) and k.size(1) == q.size(1) and k.size(3) == q.size(3) and k.size(4) == q.size(4))
    torch._check(1 <= q.size(4) <= 128)
    for w in (q_weight, k_weight):
        torch._check(w is None or (norm and w.dim() == 1 and w.size(0) == q.size(4) and w.dtype in (q.dtype, torch.float)))
    torch._check(q_weight is None or k_weight is None or q_weight.dtype == k_weight.dtype)
    torch._check(frequencies is None or (frequencies.dim() == 1 and 2 * frequencies.size(0) <= q.size(4) and frequencies.dtype == torch.double))
    torch._check(positions is None or (positions.shape == q.shape[:2] and positions.dtype == torch.int32))


@torch.library.register_fake("mamtorch_kernel_encoder::norm_rotate")
def _(q, k, q_weight, k_weight, frequencies, positions, eps, norm, interleaved):
    check_rotation(q, k, q_weight, k_weight, frequencies, positions, norm)
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))


@torch.library.register_fake("mamtorch_kernel_encoder::norm_rotate_backward")
def _(q_grad, k_grad, q, k, q_weight, k_weight, frequencies, positions, eps, norm, interleaved, want_q, want_k, want_q_weight, want_k_weight):
    check_rotation(q, k, q_weight, k_weight, frequencies, positions, norm)
    weight = q_weight if q_weight is not None else k_weight
    dtype = q.dtype if weight is None else weight.dtype
    like = [torch.empty(t.shape if w else (0,), dtype=q.dtype, device=q.device) for t, w in ((q, want_q), (k, want_k))]
    return like + [torch.empty((q.size(4) if w else 0,), dtype=dtype if w else q.dtype, device=q.device) for w in (want_q_weight, want_k_weight)]
