"""Differential attention: the difference of two softmax maps with a learned weight for each head."""
import torch
from torch import Tensor

__all__ = ["diff_attention"]

K = torch.ops.mamtorch_kernel_encoder


def diff_attention(q: Tensor, k: Tensor, v: Tensor, lam: Tensor, scale: float = None, causal: bool = False, lengths: Tensor = None,
                   starts: Tensor = None, key_mask: Tensor = None) -> Tensor:
    """``(softmax(scale q[..., 0, :] k[..., 0, :]^T) - lam softmax(scale q[..., 1, :] k[..., 1, :]^T)) v`` for each head.

    q (batch, queries, heads, 2, d), k (batch, keys, key heads, 2, d), v (batch, keys, key heads, dv), lam (heads): float32, bfloat16 or
    float16 (lam of that type or float32); d up to 128, dv up to 256; consecutive heads share a key head.  Any strides: projections
    and caches are taken as they are where the last dimension is contiguous.  Returns (batch, queries, heads, dv).

    scale: default d ** -0.5.
    lengths: int32 (batch), how many of a request's keys there are; what a cache holds past them is not used.
    key_mask: bool (batch, keys), False for keys that no query sees.
    causal: query i sees keys j <= i + starts[batch]; starts: int32 (batch), the place of the first query among the keys, by default
    keys - queries.
    A query that sees no key gives zeros.  Where a causal call's keys or values hold NaN or infinities, the queries before them may be reached
    too.  Softmaxes and sums are float32.  In 16-bit types what enters a second product is rounded to the type: the
    probabilities beside v and, in the backward pass, beside the incoming gradient, and the gradients of the scores.  Training keeps two float32
    tensors of the result's shape (float32 operands: one) until the backward pass."""
    return K.diff_attention.default(q, k, v, lam, float(q.shape[-1] ** -0.5 if scale is None else scale), bool(causal), lengths, starts,
                                    key_mask, False)[0]


def _check(q, k, v, lam):
    torch._check(q.dim() == 5 and k.dim() == 5 and v.dim() == 4 and q.size(3) == 2 and k.size(3) == 2)
    torch._check(k.size(0) == q.size(0) and v.shape[:3] == k.shape[:3] and k.size(4) == q.size(4))
    torch._check(q.dtype == k.dtype and q.dtype == v.dtype and lam.dtype in (q.dtype, torch.float))
    torch._check(lam.dim() == 1 and lam.size(0) == q.size(2))


@torch.library.register_fake("mamtorch_kernel_encoder::diff_attention")
def _(q, k, v, lam, scale, causal, lengths, starts, key_mask, with_sums):
    _check(q, k, v, lam)
    b, n, h = q.shape[:3]
    shape = (b, n, h, v.size(3))
    return [torch.empty(shape, dtype=q.dtype, device=q.device),
            torch.empty((1 if q.dtype == torch.float else 2,) + shape if with_sums else (0,), dtype=torch.float, device=q.device),
            torch.empty((2, b, h, n) if with_sums else (0,), dtype=torch.float, device=q.device)]


@torch.library.register_fake("mamtorch_kernel_encoder::diff_attention_backward")
def _(grad, q, k, v, lam, out, kept, lse, scale, causal, lengths, starts, key_mask, want_q, want_kv, want_lam):
    _check(q, k, v, lam)
    torch._check(grad.shape == out.shape and kept.shape[1:] == out.shape)
    wanted = ((q, want_q), (k, want_kv), (v, want_kv), (lam, want_lam))
    return [torch.empty(t.shape if w else (0,), dtype=t.dtype, device=t.device) for t, w in wanted]
