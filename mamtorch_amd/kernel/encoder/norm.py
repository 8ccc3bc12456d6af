"""Layer norm, and the join of a layer's halves: residual + dropout, then the norm of the next half."""
import torch
from torch import Tensor

from .dropout import default_scale, word

__all__ = ["layer_norm", "add_dropout_layer_norm"]

K = torch.ops.mamtorch_kernel_encoder


def layer_norm(x: Tensor, weight: Tensor = None, bias: Tensor = None, eps: float = 1e-5) -> Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of ``x`` (float32, bfloat16 or float16), with the biased
    variance.  ``weight`` and ``bias`` are of x's type or float32, or None.  Statistics and sums are float32; gradients do not
    depend on the order in which the GPU happens to work."""
    return K.layer_norm.default(x, weight, bias, float(eps), False)[0]


def add_dropout_layer_norm(x: Tensor, residual: Tensor, weight: Tensor = None, bias: Tensor = None, p: float = 0.0, seed: int = 0,
                           offset: int = 0, eps: float = 1e-5, step: Tensor = None):
    """``(layer_norm(s), s)`` of ``s = residual + dropout(x, p, seed, offset)``, in one pass over the operands.  The norm is that of
    ``s`` as it is returned, rounded to its type."""
    y, s = K.add_dropout_layer_norm.default(x, residual, weight, bias, float(p), default_scale(p), word(seed), word(offset), float(eps), step,
                                            False)[:2]
    return y, s


def _check_weight(x, t):
    torch._check(t is None or (t.dim() == 1 and t.size(0) == x.size(-1) and t.dtype in (x.dtype, torch.float)))


def _stats(x, wanted):
    rows = (x.numel() // x.size(-1) if x.size(-1) else 0) if wanted else 0
    return [torch.empty((rows,), dtype=torch.float, device=x.device) for _ in range(2)]


def _vector(x, wanted, is_float):
    return torch.empty((x.size(-1) if wanted else 0,), dtype=torch.float if is_float and wanted else x.dtype, device=x.device)


@torch.library.register_fake("mamtorch_kernel_encoder::layer_norm")
def _(x, weight, bias, eps, with_stats):
    torch._check(x.dim() >= 1)
    _check_weight(x, weight)
    _check_weight(x, bias)
    return [torch.empty(x.shape, dtype=x.dtype, device=x.device)] + _stats(x, with_stats)


@torch.library.register_fake("mamtorch_kernel_encoder::layer_norm_backward")
def _(grad, x, weight, mean, rstd, want_x, want_weight, want_bias, weight_is_float):
    torch._check(grad.shape == x.shape)
    is_float = weight.dtype == torch.float if weight is not None else weight_is_float
    dx = torch.empty(x.shape if want_x else (0,), dtype=x.dtype, device=x.device)
    return [dx, _vector(x, want_weight, is_float), _vector(x, want_bias, is_float)]


@torch.library.register_fake("mamtorch_kernel_encoder::add_dropout_layer_norm")
def _(x, residual, weight, bias, p, scale, seed, offset, eps, step, with_stats):
    torch._check(x.dim() >= 1 and residual.shape == x.shape and residual.dtype == x.dtype)
    _check_weight(x, weight)
    _check_weight(x, bias)
    return [torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(2)] + _stats(x, with_stats)


@torch.library.register_fake("mamtorch_kernel_encoder::add_dropout_layer_norm_backward")
def _(grad, grad_sum, s, weight, mean, rstd, p, scale, seed, offset, step, want_x, want_residual, want_weight, want_bias, weight_is_float):
    torch._check(grad.shape == s.shape)
    is_float = weight.dtype == torch.float if weight is not None else weight_is_float
    like = [torch.empty(s.shape if wanted else (0,), dtype=s.dtype, device=s.device) for wanted in (want_x, want_residual)]
    return like + [_vector(s, want_weight, is_float), _vector(s, want_bias, is_float)]
