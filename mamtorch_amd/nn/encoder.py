"""What an encoder layer has beside its MAM layers, and the layer: layer norm, dropout without a stored mask, differential attention with its
cache, and ``MAMEncoderLayer``, in which they run together with ``FullyConnected``.

The reference swaps the two Linear layers of a ViT's encoder layer for MAM layers and leaves the rest to its model library
(examples/vitb16_imagenet1k/utils.py:50-77); here the rest is the framework's operators too (``mamtorch.kernel.encoder``).
"""
import math

import torch
from torch import Tensor, nn

from ..kernel import encoder as K
from .fullyconnected import FullyConnected, check_counted

__all__ = ["LayerNorm", "Dropout", "DiffAttention", "DiffAttentionCache", "MAMEncoderLayer"]


class LayerNorm(nn.Module):
    """Layer norm over the last dimension; parameters and state as ``torch.nn.LayerNorm`` has them."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None):
        super().__init__()
        self.features, self.eps = features, eps
        self.weight = nn.Parameter(torch.ones(features, device=device, dtype=dtype))
        if bias:
            self.bias = nn.Parameter(torch.zeros(features, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def forward(self, x: Tensor) -> Tensor:
        return K.layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.features}, eps={self.eps}, bias={self.bias is not None}"


class Dropout(nn.Module):
    """Dropout whose mask is formed from (seed, number of the training call) where it is needed.  The number of calls is part of the module's
    state, so that a training run that is taken up again draws on.

    seed: modules of one model need seeds of their own, or they drop the same elements.  By default each takes one from torch's generator, when it is
    made (with p = 0, when it is first needed); that one is part of the state too, and a module whose seed was not given takes it up with the state.

    step: one int64 element on the GPU, by which the mask is numbered instead of by calls.  The training loop advances it between steps, after the
    backward pass; every call of a step draws the same mask, so what is computed again in the backward pass (activation checkpointing) and the replays
    of a captured step are right.  The word is the loop's to save, and a copy of the module has a copy of it.  Numbered by calls, a training call in a backward pass, under capture or in a DataParallel replica is an error: it would
    draw another mask than the one whose gradient is wanted, or the same one in every step; and compiled code leaves its graph at every mask, which ``fullgraph``
    refuses."""

    # for modules that were saved whole before they had these
    step, seed_given = None, True

    def __init__(self, p: float = 0.5, seed: int = None, step: Tensor = None):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError(f"p must be between 0 and 1, got {p}")
        self.p, self.seed, self.seed_given, self.step, self.calls = p, seed, seed is not None, step, 0
        if p > 0:
            self._need_seed()

    def _need_seed(self) -> None:
        if self.seed is None:
            self.seed = int(torch.randint(2 ** 63 - 1, (), device="cpu"))

    def next_offset(self) -> int:
        """Offset of this training call's mask (to which ``step`` is added where there is one), under ``seed``."""
        self._need_seed()
        if self.step is not None:
            return 0
        check_counted(self, "step")
        self.calls += 1
        return self.calls - 1

    def forward(self, x: Tensor, residual: Tensor = None) -> Tensor:
        if not self.training or self.p == 0:
            return x if residual is None else residual + x
        offset = self.next_offset()
        return K.dropout(x, self.p, self.seed, offset, residual, step=self.step)

    def get_extra_state(self):
        return {"calls": self.calls, "seed": self.seed}

    def set_extra_state(self, state):
        self.calls = int(state["calls"])
        if not self.seed_given and state.get("seed") is not None:
            self.seed = int(state["seed"])

    def extra_repr(self) -> str:
        return f"p={self.p}, seed={self.seed}"


class DiffAttentionCache:
    """Keys and values of up to ``most`` tokens for each request, and how many each has: as many for every request, since an append puts the same number
    behind each."""

    def __init__(self, batch: int, most: int, kv_heads: int, head_size: int, value_size: int, device=None, dtype=None):
        self.most = most
        self.k = torch.empty(batch, most, kv_heads, 2, head_size, device=device, dtype=dtype)
        self.v = torch.empty(batch, most, kv_heads, value_size, device=device, dtype=dtype)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        self.filled = 0                     # most tokens of a request, on the host

    def append(self, k: Tensor, v: Tensor) -> Tensor:
        """Puts k (batch, n, ...) and v behind what there is; returns the places of the first of them."""
        n = k.shape[1]
        if k.shape[0] != self.k.shape[0]:
            raise ValueError(f"the cache is for {self.k.shape[0]} requests, got {k.shape[0]}")
        if self.filled + n > self.most:
            raise ValueError(f"the cache holds {self.most} tokens: {self.filled} and {n} more do not fit")
        starts = self.lengths.clone()
        at = starts.long()[:, None] + torch.arange(n, device=starts.device)
        rows = torch.arange(k.shape[0], device=starts.device)[:, None]
        self.k[rows, at] = k
        self.v[rows, at] = v
        self.lengths += n
        self.filled += n
        return starts


class DiffAttention(nn.Module):
    """Differential attention after T. Ye et al., "Differential Transformer", 2024: each head's map is the difference of two softmaxes, the second one weighted
    with lambda = exp(q1 . k1) - exp(q2 . k2) + lambda_init from learned vectors, each head's output is normalised by itself and scaled with
    1 - lambda_init.  ``heads`` heads of two maps of size hidden / (2 heads) and values of size hidden / heads, over ``kv_heads`` key heads.

    Not as there: lambda is a head's own, not the layer's, and a head's output goes through a layer norm with mean and bias, not a root-mean-square norm, so weights do
    not carry over."""

    def __init__(self, hidden: int, heads: int, kv_heads: int = None, depth: int = 1, causal: bool = False, bias: bool = True, eps: float = 1e-5,
                 device=None, dtype=None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if hidden % (2 * heads):
            raise ValueError(f"hidden ({hidden}) must be a multiple of twice the heads ({heads})")
        if heads % kv_heads:
            raise ValueError(f"kv_heads ({kv_heads}) must divide heads ({heads})")
        kwargs = {"device": device, "dtype": dtype}
        self.hidden, self.heads, self.kv_heads, self.causal = hidden, heads, kv_heads, causal
        self.head_size, self.value_size = hidden // (2 * heads), hidden // heads
        self.lambda_init = 0.8 - 0.6 * math.exp(-0.3 * (depth - 1))
        self.query = nn.Linear(hidden, heads * 2 * self.head_size, bias=bias, **kwargs)
        self.key = nn.Linear(hidden, kv_heads * 2 * self.head_size, bias=bias, **kwargs)
        self.value = nn.Linear(hidden, kv_heads * self.value_size, bias=bias, **kwargs)
        self.output = nn.Linear(hidden, hidden, bias=bias, **kwargs)
        self.lambda_vectors = nn.Parameter(0.1 * torch.randn(4, heads, self.head_size, **kwargs))
        self.norm = LayerNorm(self.value_size, eps, **kwargs)

    def lambdas(self) -> Tensor:
        q1, k1, q2, k2 = self.lambda_vectors.float()
        return torch.exp((q1 * k1).sum(-1)) - torch.exp((q2 * k2).sum(-1)) + self.lambda_init

    def cache(self, batch: int, most: int) -> DiffAttentionCache:
        """A cache for this module's keys and values, in the type that they have where it is made (under autocast, autocast's)."""
        weight = self.key.weight
        dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else weight.dtype
        return DiffAttentionCache(batch, most, self.kv_heads, self.head_size, self.value_size, weight.device, dtype)

    def forward(self, x: Tensor, lengths: Tensor = None, key_mask: Tensor = None, cache: DiffAttentionCache = None) -> Tensor:
        """x (batch, tokens, hidden).  With a cache, x's tokens are put behind it and see what is there (up to themselves where the module is
        causal); lengths and key_mask (see ``kernel.encoder.diff_attention``) are for calls without one."""
        b, n = x.shape[:2]
        q = self.query(x).view(b, n, self.heads, 2, self.head_size)
        k = self.key(x).view(b, n, self.kv_heads, 2, self.head_size)
        v = self.value(x).view(b, n, self.kv_heads, self.value_size)
        starts = None
        if cache is not None:
            if lengths is not None or key_mask is not None:
                raise ValueError("a cache has lengths of its own")
            starts = cache.append(k, v)
            k, v, lengths = cache.k[:, :cache.filled], cache.v[:, :cache.filled], cache.lengths
        elif self.causal:
            starts = torch.zeros(b, device=x.device, dtype=torch.int32)
        out = K.diff_attention(q, k, v, self.lambdas(), causal=self.causal, lengths=lengths, starts=starts if self.causal else None, key_mask=key_mask)
        out = self.norm(out) * (1 - self.lambda_init)
        return self.output(out.reshape(b, n, self.hidden))


class MAMEncoderLayer(nn.Module):
    """A pre-norm encoder layer: x + dropout(attention(norm(x))), then the same of the MAM MLP (FullyConnected -> GELU -> FullyConnected).
    The sum between the halves, its dropout and the second norm are one operator.  ViT-B/16: hidden 768, intermediate 3072, 6 heads of two maps.
    Parameters and x are float32, as the MAM layers are; under autocast the attention runs in 16 bits between them.

    seed: of the two dropouts, each under a key formed from it and from depth; layers of one depth need seeds of their own, by default drawn as ``Dropout``
    does.  ``wdrop_seed`` is likewise the two weights'.  step: what numbers the masks instead of calls (see ``Dropout``), those of the ``FullyConnected`` layers' weights too.  Further keyword arguments go to
    the ``FullyConnected`` layers."""

    def __init__(self, hidden: int = 768, intermediate: int = 3072, heads: int = 6, kv_heads: int = None, depth: int = 1, causal: bool = False,
                 p: float = 0.0, seed: int = None, eps: float = 1e-5, device=None, dtype=None, step: Tensor = None, **fc_kwargs):
        super().__init__()
        kwargs = {"device": device, "dtype": dtype}
        fc_kwargs.setdefault("wdrop_step", step)
        seeds = (None, None) if seed is None else (2 * seed + (depth - 1 << 32), 2 * seed + 1 + (depth - 1 << 32))
        wdrop_seed = fc_kwargs.pop("wdrop_seed", None)      # high bits: no key of a weight is a dropout's or the other weight's
        wdrop_seeds = (None, None) if wdrop_seed is None else tuple(wdrop_seed + (depth - 1 << 32) + (n << 61) for n in (1, 2))
        self.norm1 = LayerNorm(hidden, eps, **kwargs)
        self.attention = DiffAttention(hidden, heads, kv_heads, depth, causal, **kwargs)
        self.dropout1 = Dropout(p, seeds[0], step)
        self.norm2 = LayerNorm(hidden, eps, **kwargs)
        self.intermediate = FullyConnected(hidden, intermediate, wdrop_seed=wdrop_seeds[0], **kwargs, **fc_kwargs)
        self.act = nn.GELU()
        self.output = FullyConnected(intermediate, hidden, wdrop_seed=wdrop_seeds[1], **kwargs, **fc_kwargs)
        self.dropout2 = Dropout(p, seeds[1], step)

    def vcon_step(self) -> None:
        self.intermediate.vcon_step()
        self.output.vcon_step()

    def forward(self, x: Tensor, lengths: Tensor = None, key_mask: Tensor = None, cache: DiffAttentionCache = None) -> Tensor:
        a = self.attention(self.norm1(x), lengths, key_mask, cache).to(x.dtype)      # 16 bits under autocast
        drop, norm = self.dropout1, self.norm2
        p = drop.p if drop.training else 0.0
        offset = drop.next_offset() if p else 0
        y, s = K.add_dropout_layer_norm(a, x, norm.weight, norm.bias, p, drop.seed if p else 0, offset, norm.eps, step=drop.step if p else None)
        return self.dropout2(self.output(self.act(self.intermediate(y))), s)
