"""A cache in pages: its bookkeeping on the device, what puts keys and values into it, and differential attention over it.

Keys k_pages (pages, key heads, page size, 2, d) and values v_pages (pages, key heads, page size, dv), contiguous, page size a multiple of 16.  table (batch, slots):
the page of a request's tokens slot * page size .., -1 where there is none; lengths (batch): its tokens; refs (pages): how many requests hold a page, 0 where it is
free.  All three are int32; the calls that change them do so in place, on the current stream, and nothing waits for the GPU, so that a whole step can be captured.  At most 4096
requests.  One table may serve the pages of many layers.
"""
import torch
from torch import Tensor

from .rotary import TYPES, check_rotation

__all__ = ["pages_extend", "pages_fork", "pages_trim", "pages_copy", "pages_compact", "draft_tree", "norm_rotate_append", "diff_attention_pages"]

K = torch.ops.mamtorch_kernel_encoder


def pages_extend(table: Tensor, lengths: Tensor, refs: Tensor, counts: Tensor, page_size: int):
    """Room for ``counts`` (batch, int32) tokens behind each request's: ``(granted, copies)``.

    Pages are the free ones of lowest number, in the requests' order.  A begun last page that other requests hold too is given up for a new one, but by the last request that
    holds it; copies (batch, 2) names the page and the new one, for ``pages_copy``, or is -1.  granted (batch): a request's count, or 0 where the free pages or the table's slots do
    not reach: that request is left as it was, and so are those behind it that need pages,
    or that would write to a page which it was to give up."""
    return K.pages_extend.default(table, lengths, refs, counts, int(page_size))


def pages_fork(table: Tensor, lengths: Tensor, refs: Tensor, sources: Tensor, page_size: int) -> None:
    """Request i goes on from what request ``sources[i]`` (batch, int32) was before the call, whose pages both hold then; room behind its tokens is given back.
    -1, or any number that is no request, leaves it empty."""
    K.pages_fork.default(table, lengths, refs, sources, int(page_size))


def pages_trim(table: Tensor, lengths: Tensor, refs: Tensor, ends: Tensor, page_size: int) -> None:
    """Requests have ``ends`` (batch, int32) tokens, more or fewer than before but no more than their pages hold; pages behind are given back.  0 frees a request."""
    K.pages_trim.default(table, lengths, refs, ends, int(page_size))


def pages_copy(k_pages: Tensor, v_pages: Tensor, copies: Tensor) -> None:
    """Copies page ``copies[i, 0]`` to page ``copies[i, 1]`` (int32), but where one of them is -1.  No page is written that another pair reads or writes."""
    K.pages_copy.default(k_pages, v_pages, copies)


def pages_compact(k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, path: Tensor, counts: Tensor = None) -> None:
    """Takes over drafted tokens: token ``lengths + path[:, i]`` becomes token ``lengths + i``, for i below ``counts`` (batch, int32; all by default).  ``path`` (batch, n), int32,
    ascends in each row; from an entry on that does not, a request's tokens stay.  Lengths are not changed (``pages_trim``)."""
    K.pages_compact.default(k_pages, v_pages, table, lengths, path, counts)


def draft_tree(parents: Tensor, lengths: Tensor = None):
    """``(masks, positions)`` of trees of up to 64 drafted tokens: parents (batch, n), int32, the token that one follows, which stands before it, or -1.  masks (batch, n),
    int64: bit j of a token's mask is set where it sees token j, itself or one above it; positions (batch, n), int32: ``lengths`` plus how many are above it."""
    return K.draft_tree.default(parents, lengths)


def norm_rotate_append(q: Tensor, k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, q_weight: Tensor = None,
                       k_weight: Tensor = None, frequencies: Tensor = None, positions: Tensor = None, eps: float = 1e-6, norm: bool = True,
                       interleaved: bool = False, counts: Tensor = None) -> Tensor:
    """``norm_rotate`` of new tokens behind those of the cache: returns the queries; the keys, and the values v (batch, tokens, key heads, dv), go to the pages of tokens
    ``lengths + i``, for i below ``counts`` (batch, int32; all by default) and where the request has a page.  positions: by default ``lengths + i``.  Lengths are not changed.
    norm False and no frequencies: keys and values as they are.  No gradient."""
    return K.norm_rotate_append.default(q, k, v, k_pages, v_pages, table, lengths, counts, q_weight, k_weight, frequencies, positions, float(eps), bool(norm),
                                        bool(interleaved))


def diff_attention_pages(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, lam: Tensor, scale: float = None,
                         counts: Tensor = None, masks: Tensor = None) -> Tensor:
    """``diff_attention`` of new tokens q (batch, n, heads, 2, d), whose keys and values stand behind the cache's ``lengths`` tokens in the pages already: each sees all tokens of the
    cache and, of the new ones, those up to itself or, where there are masks (batch, n <= 64; int64), those whose bits are set.

    counts (batch, int32): how many of the n tokens a request has, all by default.  A token beyond, or one that sees nothing, gives zeros.  Tokens for which a request has no
    page are not seen.  Softmaxes and sums are float32; in 16-bit types the probabilities beside v are rounded to the type, those of the first map in two parts, whatever the number of tokens.
    What pages hold behind a request's tokens may be anything; NaN or infinities among the new tokens' values may reach those before them, and beside
    them in the tree.  No gradient."""
    return K.diff_attention_pages.default(q, k_pages, v_pages, table, lengths, lam, float(q.shape[-1] ** -0.5 if scale is None else scale), counts, masks)


# What the operators refuse by shapes and types is refused under tracing too.
def _check_vector(t, n):
    torch._check(t is None or (t.dim() == 1 and t.size(0) == n and t.dtype == torch.int32))


def _check_pages(k_pages, v_pages):
    torch._check(k_pages.dim() == 5 and v_pages.dim() == 4 and k_pages.size(3) == 2 and k_pages.dtype == v_pages.dtype and k_pages.dtype in TYPES)
    torch._check(k_pages.shape[:3] == v_pages.shape[:3])
    torch._check(k_pages.size(2) >= 16 and k_pages.size(2) % 16 == 0)
    torch._check(1 <= k_pages.size(4) <= 128 and 1 <= v_pages.size(3) <= 256)


def _check_table(table, *vectors):
    torch._check(table.dim() == 2 and table.dtype == torch.int32)
    for t in vectors:
        _check_vector(t, table.size(0))


def _check_book(table, lengths, refs, more, page_size):
    _check_table(table, lengths, more)
    torch._check(refs.dim() == 1 and refs.dtype == torch.int32)
    torch._check(page_size >= 16 and page_size % 16 == 0 and table.size(0) <= 4096)


@torch.library.register_fake("mamtorch_kernel_encoder::pages_extend")
def _(table, lengths, refs, counts, page_size):
    _check_book(table, lengths, refs, counts, page_size)
    return table.new_empty((table.size(0),)), table.new_empty((table.size(0), 2))


@torch.library.register_fake("mamtorch_kernel_encoder::pages_fork")
def _(table, lengths, refs, sources, page_size):
    _check_book(table, lengths, refs, sources, page_size)


@torch.library.register_fake("mamtorch_kernel_encoder::pages_trim")
def _(table, lengths, refs, ends, page_size):
    _check_book(table, lengths, refs, ends, page_size)


@torch.library.register_fake("mamtorch_kernel_encoder::pages_copy")
def _(k_pages, v_pages, copies):
    _check_pages(k_pages, v_pages)
    torch._check(copies.dim() == 2 and copies.size(1) == 2 and copies.dtype == torch.int32)


@torch.library.register_fake("mamtorch_kernel_encoder::pages_compact")
def _(k_pages, v_pages, table, lengths, path, counts):
    _check_pages(k_pages, v_pages)
    _check_table(table, lengths, counts)
    torch._check(path.dim() == 2 and path.size(0) == table.size(0) and path.dtype == torch.int32)


@torch.library.register_fake("mamtorch_kernel_encoder::draft_tree")
def _(parents, lengths):
    torch._check(parents.dim() == 2 and parents.size(1) <= 64 and parents.dtype == torch.int32)
    _check_vector(lengths, parents.size(0))
    return parents.new_empty(parents.shape, dtype=torch.long), parents.new_empty(parents.shape)


@torch.library.register_fake("mamtorch_kernel_encoder::norm_rotate_append")
def _(q, k, v, k_pages, v_pages, table, lengths, counts, q_weight, k_weight, frequencies, positions, eps, norm, interleaved):
    check_rotation(q, k, q_weight, k_weight, frequencies, positions, norm)
    _check_pages(k_pages, v_pages)
    _check_table(table, lengths, counts)
    torch._check(q.size(3) == 2 and q.size(0) == table.size(0) and v.dtype == q.dtype and k_pages.dtype == q.dtype)
    torch._check(v.dim() == 4 and v.shape[:3] == k.shape[:3])
    torch._check(k_pages.size(1) == k.size(2) and k_pages.size(4) == k.size(4) and v_pages.size(3) == v.size(3))
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


@torch.library.register_fake("mamtorch_kernel_encoder::diff_attention_pages")
def _(q, k_pages, v_pages, table, lengths, lam, scale, counts, masks):
    _check_pages(k_pages, v_pages)
    _check_table(table, lengths, counts)
    torch._check(q.dim() == 5 and q.size(3) == 2 and q.size(4) == k_pages.size(4) and q.size(0) == table.size(0) and q.dtype == k_pages.dtype)
    torch._check(q.size(2) == 0 or (k_pages.size(1) > 0 and q.size(2) % k_pages.size(1) == 0))
    torch._check(lam.dim() == 1 and lam.size(0) == q.size(2) and lam.dtype in (q.dtype, torch.float))
    torch._check(0 < scale <= 1e30)
    torch._check(masks is None or (q.size(1) <= 64 and masks.shape == q.shape[:2] and masks.dtype == torch.long))
    return torch.empty((*q.shape[:3], v_pages.size(3)), dtype=q.dtype, device=q.device)
