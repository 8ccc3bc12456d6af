"""What an encoder layer has beside its MAM layers, and the layer: layer norm, dropout without a stored mask, differential attention with its
caches, and ``MAMEncoderLayer``, in which they run together with ``FullyConnected``.

The reference swaps the two Linear layers of a ViT's encoder layer for MAM layers and leaves the rest to its model library
(examples/vitb16_imagenet1k/utils.py:50-77); here the rest is the framework's operators too (``mamtorch.kernel.encoder``).
"""
import math

import torch
from torch import Tensor, nn

from ..kernel import encoder as K
from .fullyconnected import FullyConnected, check_counted

__all__ = ["LayerNorm", "Dropout", "DiffAttention", "DiffAttentionCache", "DiffAttentionPages", "PageTable", "MAMEncoderLayer"]


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


class PageTable:
    """Which pages of a cache up to ``batch`` requests hold, of ``pages`` pages of ``page_size`` tokens each and up to ``most`` tokens a request: one for all layers of a model, each of
    which has the pages themselves (``DiffAttention.pages``).  On the device: nothing here waits for the GPU, and a step may be captured.

    A step of a server is ``begin``, the model on the new tokens under ``torch.no_grad()``, ``accept``.  In between, ``fork`` and ``trim`` change which requests there are.  Requests have
    tokens and counts of their own; one that has none in a step is given a count of 0."""

    def __init__(self, batch: int, pages: int, page_size: int = 64, most: int = None, device=None):
        if page_size < 16 or page_size % 16:
            raise ValueError(f"a page holds a multiple of 16 tokens, got {page_size}")
        self.batch, self.pages, self.page_size = batch, pages, page_size
        slots = pages if most is None else -(-most // page_size)
        self.table = torch.full((batch, slots), -1, device=device, dtype=torch.int32)
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        self.refs = torch.zeros(pages, device=device, dtype=torch.int32)
        self.caches = []
        self.granted = self.masks = self.positions = None       # of the step that has begun

    def _vector(self, value) -> Tensor:
        if isinstance(value, Tensor):
            return value.to(torch.int32)
        return torch.full((self.batch,), value, device=self.lengths.device, dtype=torch.int32)

    def begin(self, counts=None, parents: Tensor = None) -> Tensor:
        """Room for ``counts`` new tokens behind each request's (a number, or int32 (batch)), or for trees of drafted tokens, ``parents`` (batch, n) as
        ``kernel.encoder.draft_tree`` takes them, or for the first ``counts`` tokens of those.  Returns how many tokens each request has room for: its count or, where the pages do not reach, 0, and then its tokens
        are not written and give zeros."""
        if (counts is None) and (parents is None):
            raise ValueError("a step has counts or parents")
        self.masks = self.positions = None
        if parents is None:
            counts = self._vector(counts)
        else:
            n = parents.shape[1]
            counts = self._vector(n) if counts is None else self._vector(counts).clamp(max=n)
        self.granted, copies = K.pages_extend(self.table, self.lengths, self.refs, counts, self.page_size)
        # whatever the step: how long pages stay in common after a fork, and whether a replayed graph held one, the device alone knows.  (4 to 5 us a layer where there is
        # nothing to copy: one token of 64 requests through 12 layers of 768 takes 3.20 ms, 3.11 without.)
        for cache in self.caches:
            K.pages_copy(cache.k, cache.v, copies)
        if parents is not None:
            self.masks, self.positions = K.draft_tree(parents, self.lengths)
        return self.granted

    def accept(self, path: Tensor = None, counts=None) -> None:
        """Takes over the new tokens of the step: the first ``counts`` of each request (a number, or int32 (batch); by default all that it had room for) or, with ``path``
        (batch, n), int32, those that it names, in ascending order, up to an entry that does not ascend or names none of them.  No more than there was room for; other new
        tokens are forgotten."""
        if self.granted is None:
            raise ValueError("no step has begun")
        counts = self.granted if counts is None else torch.minimum(self._vector(counts).clamp(min=0), self.granted)
        if path is not None:
            counts = torch.minimum(counts, self._named(path))
            for cache in self.caches:
                K.pages_compact(cache.k, cache.v, self.table, self.lengths, path, counts)
        self.trim(self.lengths + counts)

    def _named(self, path: Tensor) -> Tensor:
        """How many entries of each request's path name tokens that it had room for, in ascending order."""
        n = path.shape[1]
        if n == 0:
            return torch.zeros_like(self.granted)
        ok = (path > nn.functional.pad(path, (1, 0), value=-1)[:, :-1]) & (path < self.granted[:, None])
        # a running minimum, not a reduction: one over many blocks would clear its memory by a node that a graph must not hold
        return torch.where(ok, n, torch.arange(n, device=path.device, dtype=torch.int32)).cummin(1).values[:, -1]

    def trim(self, ends) -> None:
        """Requests end at ``ends`` (a number, or int32 (batch)); 0 frees a request."""
        K.pages_trim(self.table, self.lengths, self.refs, self._vector(ends), self.page_size)
        self.granted = self.masks = self.positions = None

    def fork(self, sources: Tensor) -> None:
        """Request i goes on from what request ``sources[i]`` (int32) was; -1 frees it."""
        K.pages_fork(self.table, self.lengths, self.refs, sources, self.page_size)
        self.granted = self.masks = self.positions = None


class DiffAttentionPages:
    """A layer's keys and values in the pages of a ``PageTable``."""

    def __init__(self, table: PageTable, kv_heads: int, head_size: int, value_size: int, device=None, dtype=None):
        self.table = table
        self.k = torch.empty(table.pages, kv_heads, table.page_size, 2, head_size, device=device, dtype=dtype)
        self.v = torch.empty(table.pages, kv_heads, table.page_size, value_size, device=device, dtype=dtype)
        table.caches.append(self)

    def append(self, q: Tensor, k: Tensor, v: Tensor, q_weight: Tensor = None, k_weight: Tensor = None, frequencies: Tensor = None, eps: float = 1e-6,
               norm: bool = True) -> Tensor:
        """Puts the step's keys, normed and turned, and values behind what there is; returns the queries, normed and turned."""
        t = self._begun()
        return K.norm_rotate_append(q, k, v, self.k, self.v, t.table, t.lengths, q_weight, k_weight, frequencies, t.positions, eps, norm, counts=t.granted)

    def attend(self, q: Tensor, lam: Tensor) -> Tensor:
        """Differential attention of the step's queries over what there is and the step's own tokens, up to themselves or up their tree."""
        t = self._begun()
        return K.diff_attention_pages(q, self.k, self.v, t.table, t.lengths, lam, counts=t.granted, masks=t.masks)

    def _begun(self) -> PageTable:
        if self.table.granted is None:
            raise ValueError("no step has begun: call the table's begin()")
        return self.table


def _place_after_load(module: "DiffAttention", keys) -> None:
    # parameters that are assigned may stand on another device than the ones before
    module._place_frequencies()


class DiffAttention(nn.Module):
    """Differential attention after T. Ye et al., "Differential Transformer", 2024: each head's map is the difference of two softmaxes, the second one weighted
    with lambda = exp(q1 . k1) - exp(q2 . k2) + lambda_init from learned vectors, each head's output is normalised by itself and scaled with
    1 - lambda_init.  ``heads`` heads of two maps of size hidden / (2 heads) and values of size hidden / heads, over ``kv_heads`` key heads.

    Not as there: lambda is a head's own, not the layer's, and a head's output goes through a layer norm with mean and bias, not a root-mean-square norm, so weights do
    not carry over.

    qk_norm: each head's queries and keys are normalised by their root mean square, with weights ``query_norm`` and ``key_norm``.  rotary: how many elements of a head turn by
    the token's place (an even number; True: all of them), pair i by ``base ** (-2 i / rotary)`` a place; places count from a request's first token."""

    # for modules that were saved whole before they had these
    qk_norm, rotary, base, qk_eps, frequencies = False, 0, 10000.0, 1e-6, None

    def __init__(self, hidden: int, heads: int, kv_heads: int = None, depth: int = 1, causal: bool = False, bias: bool = True, eps: float = 1e-5,
                 device=None, dtype=None, qk_norm: bool = False, rotary: int = 0, base: float = 10000.0):
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
        self.qk_norm, self.rotary, self.base, self.qk_eps = qk_norm, self.head_size if rotary is True else int(rotary), base, 1e-6
        if self.rotary < 0 or self.rotary % 2 or self.rotary > self.head_size:
            raise ValueError(f"rotary ({rotary}) must be an even number up to the head's size ({self.head_size})")
        if qk_norm:
            self.query_norm = nn.Parameter(torch.ones(self.head_size, device=device, dtype=dtype))
            self.key_norm = nn.Parameter(torch.ones(self.head_size, device=device, dtype=dtype))
        self._place_frequencies()
        self.register_load_state_dict_post_hook(_place_after_load)

    def _place_frequencies(self) -> None:
        # no buffer: .half() and its like would round it
        device = self.query.weight.device
        if self.rotary and (self.frequencies is None or self.frequencies.device != device):
            self.frequencies = K.rotary_frequencies(self.rotary, self.base, device)

    def _apply(self, *args, **kwargs):
        super()._apply(*args, **kwargs)
        self._place_frequencies()
        return self

    def _frequencies_on(self, device: torch.device) -> Tensor:
        # a replica on another device shares the attribute
        if self.frequencies is None or self.frequencies.device == device:
            return self.frequencies
        return K.rotary_frequencies(self.rotary, self.base, device)

    def lambdas(self) -> Tensor:
        q1, k1, q2, k2 = self.lambda_vectors.float()
        return torch.exp((q1 * k1).sum(-1)) - torch.exp((q2 * k2).sum(-1)) + self.lambda_init

    def _cache_type(self) -> torch.dtype:
        return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else self.key.weight.dtype

    def cache(self, batch: int, most: int) -> DiffAttentionCache:
        """A cache for this module's keys and values, in the type that they have where it is made (under autocast, autocast's)."""
        return DiffAttentionCache(batch, most, self.kv_heads, self.head_size, self.value_size, self.key.weight.device, self._cache_type())

    def pages(self, table: PageTable) -> DiffAttentionPages:
        """This module's pages of ``table``, in that type."""
        return DiffAttentionPages(table, self.kv_heads, self.head_size, self.value_size, self.key.weight.device, self._cache_type())

    def forward(self, x: Tensor, lengths: Tensor = None, key_mask: Tensor = None, cache=None) -> Tensor:
        """x (batch, tokens, hidden).  With a ``DiffAttentionCache``, x's tokens are put behind it and see what is there (up to themselves where the module is
        causal); with ``DiffAttentionPages``, for causal modules, into the room of the step that has begun, and see what is there up to themselves or up
        their tree.  lengths and key_mask (see ``kernel.encoder.diff_attention``) are for calls without one."""
        b, n = x.shape[:2]
        if cache is not None and (lengths is not None or key_mask is not None):
            raise ValueError("a cache has lengths of its own")
        paged = isinstance(cache, DiffAttentionPages)
        if paged and not self.causal:
            raise ValueError("pages are for causal modules")
        q = self.query(x).view(b, n, self.heads, 2, self.head_size)
        k = self.key(x).view(b, n, self.kv_heads, 2, self.head_size)
        v = self.value(x).view(b, n, self.kv_heads, self.value_size)
        weights = (self.query_norm, self.key_norm) if self.qk_norm else (None, None)
        eps, frequencies = self.qk_eps if self.qk_norm else 0.0, self._frequencies_on(x.device)
        if paged:
            q = cache.append(q, k, v, *weights, frequencies, eps, self.qk_norm)
            out = cache.attend(q, self.lambdas())
        else:
            if self.qk_norm or self.rotary:
                places = None
                if self.rotary and cache is not None:
                    places = cache.lengths[:, None] + torch.arange(n, device=x.device, dtype=torch.int32)
                q, k = K.norm_rotate(q, k, *weights, frequencies, places, eps, self.qk_norm)
            starts = None
            if cache is not None:
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
    does.  ``wdrop_seed`` is likewise the two weights'.  step: what numbers the masks instead of calls (see ``Dropout``), those of the ``FullyConnected`` layers' weights too.  qk_norm, rotary,
    base: the attention's (see ``DiffAttention``, and there for caches).  Further keyword arguments go to
    the ``FullyConnected`` layers."""

    def __init__(self, hidden: int = 768, intermediate: int = 3072, heads: int = 6, kv_heads: int = None, depth: int = 1, causal: bool = False,
                 p: float = 0.0, seed: int = None, eps: float = 1e-5, device=None, dtype=None, step: Tensor = None, qk_norm: bool = False,
                 rotary: int = 0, base: float = 10000.0, **fc_kwargs):
        super().__init__()
        kwargs = {"device": device, "dtype": dtype}
        fc_kwargs.setdefault("wdrop_step", step)
        seeds = (None, None) if seed is None else (2 * seed + (depth - 1 << 32), 2 * seed + 1 + (depth - 1 << 32))
        wdrop_seed = fc_kwargs.pop("wdrop_seed", None)      # high bits: no key of a weight is a dropout's or the other weight's
        wdrop_seeds = (None, None) if wdrop_seed is None else tuple(wdrop_seed + (depth - 1 << 32) + (n << 61) for n in (1, 2))
        self.norm1 = LayerNorm(hidden, eps, **kwargs)
        self.attention = DiffAttention(hidden, heads, kv_heads, depth, causal, qk_norm=qk_norm, rotary=rotary, base=base, **kwargs)
        self.dropout1 = Dropout(p, seeds[0], step)
        self.norm2 = LayerNorm(hidden, eps, **kwargs)
        self.intermediate = FullyConnected(hidden, intermediate, wdrop_seed=wdrop_seeds[0], **kwargs, **fc_kwargs)
        self.act = nn.GELU()
        self.output = FullyConnected(intermediate, hidden, wdrop_seed=wdrop_seeds[1], **kwargs, **fc_kwargs)
        self.dropout2 = Dropout(p, seeds[1], step)

    def vcon_step(self) -> None:
        self.intermediate.vcon_step()
        self.output.vcon_step()

    def forward(self, x: Tensor, lengths: Tensor = None, key_mask: Tensor = None, cache=None) -> Tensor:
        a = self.attention(self.norm1(x), lengths, key_mask, cache).to(x.dtype)      # 16 bits under autocast
        drop, norm = self.dropout1, self.norm2
        p = drop.p if drop.training else 0.0
        offset = drop.next_offset() if p else 0
        y, s = K.add_dropout_layer_norm(a, x, norm.weight, norm.bias, p, drop.seed if p else 0, offset, norm.eps, step=drop.step if p else None)
        return self.dropout2(self.output(self.act(self.intermediate(y))), s)
