"""GPU tests of differential attention over the pages of a cache against 64 bits: sizes, trees, rows that see nothing, pages that end inside a tile, what pages hold behind
a request's tokens."""
import random

import pytest
import torch

import encoder_reference as ref
import mamtorch_amd as mt
import pages_reference as pref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
enc = mt.kernel.encoder
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _make(shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32)


def _parents(b, n, seed):
    rng = random.Random(seed)
    return [[rng.randint(-1, i - 1) for i in range(n)] for _ in range(b)]


class Case:
    def __init__(self, lengths, n, page, h, hk, d, dv, dtype, seed=0, masks=None, counts=None, scale=1.0, spare=2):
        b = len(lengths)
        used = [-(-(length + n) // page) for length in lengths]
        pages, slots = sum(used) + 5, max(used) + spare
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        self.table = _ints([[order.pop() if s < u else -1 for s in range(slots)] for u in used])
        self.lengths = _ints(lengths)
        self.counts = None if counts is None else _ints(counts)
        self.masks = masks
        self.q = _make((b, n, h, 2, d), dtype, seed + 1, scale)
        self.k, self.v = _make((pages, hk, page, 2, d), dtype, seed + 2, scale), _make((pages, hk, page, dv), dtype, seed + 3)
        self.lam = (0.2 + 0.6 * torch.rand(h, generator=torch.Generator().manual_seed(seed + 4))).to(dtype)

    def poison(self, value):
        """Everything that no request has as `value`: pages that nobody holds, and behind a request's tokens."""
        n, page = self.q.shape[1], self.k.shape[2]
        k, v = self.k.clone(), self.v.clone()
        self.k.fill_(value)
        self.v.fill_(value)
        for b in range(self.q.shape[0]):
            end = int(self.lengths[b]) + (n if self.counts is None else max(0, min(n, int(self.counts[b]))))
            for s, p in enumerate(self.table[b].tolist()):
                if p >= 0:
                    there = max(0, min(page, end - s * page))
                    self.k[p, :, :there], self.v[p, :, :there] = k[p, :, :there], v[p, :, :there]
        return self

    def run(self, q=None, lam=None, scale=None):
        on = lambda t: None if t is None else t.to(DEV)                                     # noqa: E731
        return enc.diff_attention_pages(on(self.q) if q is None else q, on(self.k), on(self.v), on(self.table), on(self.lengths), on(self.lam if lam is None else lam), scale,
                                        on(self.counts), on(self.masks))

    def check(self, what, out=None, lam=None, scale=None):
        out = self.run(lam=lam, scale=scale) if out is None else out
        nan = lambda t: torch.where(torch.isfinite(t), t, torch.zeros((), dtype=t.dtype))   # noqa: E731  (poison is not seen)
        want = pref.PagesAttention(self.q, nan(self.k), nan(self.v), self.table, self.lengths, self.lam if lam is None else lam, scale, self.counts, self.masks)
        ref.assert_within(out, want.out, want.out_bound, what)
        return out


def _tree_masks(b, n, seed):
    return pref.bits(torch.stack([pref.tree(p) for p in _parents(b, n, seed)]))


HEADS = [(32, 64), (64, 64), (64, 128), (128, 128), (128, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d, dv", HEADS + [(33, 65), (80, 160), (1, 1), (7, 256), (128, 3)])
@pytest.mark.parametrize("n", [1, 7])
def test_heads(n, d, dv, dtype):
    Case([0, 5, 100, 333], n, 16, 4, 2, d, dv, dtype, scale=0.7).check("%d/%d" % (d, dv))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 32, 48, 64, 112, 256])
@pytest.mark.parametrize("h, hk", [(1, 1), (6, 6), (8, 2), (16, 1), (12, 4)])
def test_pages_and_groups(h, hk, page, dtype):
    lengths = [0, 1, 15, 16, 17, 31, 32, 33, page - 1, page, page + 1, 3 * page + 7, 700]
    Case(lengths, 1, page, h, hk, 64, 128, dtype, 10).check("one token")
    Case(lengths[::3], 5, page, h, hk, 64, 128, dtype, 20).check("five tokens")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 5, 16, 33, 63, 64])
@pytest.mark.parametrize("d, dv, page", [(64, 128, 16), (128, 256, 48), (32, 64, 64)])
def test_trees(d, dv, page, n, dtype):
    lengths = [0, 3, 31, 64, 250]
    Case(lengths, n, page, 4, 2, d, dv, dtype, 30, _tree_masks(5, n, n)).check("tree of %d" % n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [65, 130, 300])
@pytest.mark.parametrize("h, hk, d, dv", [(2, 2, 64, 128), (8, 2, 128, 256), (4, 1, 33, 40)])
def test_chunks_of_prompts(h, hk, d, dv, n, dtype):
    Case([0, 100, 517], n, 32, h, hk, d, dv, dtype, 40).check("chunk of %d" % n)
    Case([40, 0, 77], n, 16, h, hk, d, dv, dtype, 50, counts=[n, 3, n - 1]).check("ragged chunk of %d" % n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 6, 40])
def test_rows_that_see_nothing_are_zeros(n, dtype):
    masks = _tree_masks(5, n, 3)
    masks[0] = 0                # nothing in the cache, and nothing of the tree
    masks[1, n // 2] = 0        # one of its tokens
    masks[2] = 0                # the cache alone
    masks[3] = -1               # also bits of tokens that are not there
    case = Case([0, 0, 50, 20, 9], n, 16, 4, 2, 64, 128, dtype, 60, masks, counts=[n, n, n, n, 0])
    out = case.check("empty rows")
    assert not out[0].any() and not out[1, n // 2].any() and not out[4].any()
    assert not Case([7, 300], n, 16, 4, 2, 64, 128, dtype, 65, counts=[0, -4]).check("no tokens").any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n, tree", [(1, False), (9, True), (9, False), (70, False)])
def test_what_pages_hold_behind_the_tokens_is_not_used(n, tree, value, dtype):
    masks = _tree_masks(4, n, 5) if tree else None
    for counts in (None, [n, n - 1, 0, n // 2]):
        Case([0, 13, 64, 200], n, 48, 4, 2, 64, 128, dtype, 70, masks, counts).poison(value).check("poisoned")
        Case([0, 13, 64, 200], n, 16, 4, 4, 40, 36, dtype, 80, masks, counts).poison(value).check("poisoned, odd heads")


@pytest.mark.parametrize("dtype", TYPES)
def test_keys_of_tokens_that_are_not_seen_may_be_nan(dtype):
    # the scores of a masked key are not used, whatever they are
    masks = torch.tensor([[0b001, 0b011, 0b101]])
    case = Case([20], 3, 16, 2, 1, 64, 64, dtype, 90, masks)
    slot, at = divmod(22, 16)
    case.k[case.table[0, slot], :, at] = float("nan")
    out = case.run()
    assert torch.isfinite(out[0, :2]).all() and torch.isnan(out[0, 2]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_query_with_nan_gives_nan(dtype):
    case = Case([700, 40], 2, 16, 2, 1, 64, 64, dtype, 95)
    case.q[1, 0, 1, 0, 3] = float("nan")
    out = case.run()
    assert torch.isnan(out[1, 0, 1]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[1, 1]).all() and torch.isfinite(out[1, 0, 0]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 20])
def test_tokens_without_a_page_are_not_seen(n, dtype):
    case = Case([100, 90, 64, 10], n, 16, 4, 2, 64, 128, dtype, 100)
    case.table[0, 2] = -1
    case.table[1, 0] = case.k.shape[0]          # no page of these
    case.table[2] = -1
    case.table[3, 0] = 2 ** 31 - 1
    case.check("holes")
    case = Case([100, 90], n, 16, 4, 2, 64, 128, dtype, 110, spare=0)
    case.lengths = _ints([2 ** 31 - 1, -2 ** 31])                   # more than the slots hold; fewer than none
    case.check("lengths that cannot be")


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_that_rise_late_and_large_ones(dtype):
    case = Case([2000], 2, 64, 4, 2, 64, 128, dtype, 120, scale=0.05)
    last = case.table[0, 1900 // 64]
    case.k[last, :, 1900 % 64] *= 200
    case.check("a late maximum")
    case = Case([500, 3], 4, 16, 4, 2, 64, 64, dtype, 130, scale=6.0)
    case.check("large scores")
    case.check("a scale", scale=0.02)


@pytest.mark.parametrize("dtype", TYPES)
def test_lambdas(dtype):
    case = Case([333, 20], 3, 32, 4, 2, 64, 128, dtype, 140)
    for lam in (torch.zeros(4), torch.tensor([-3.0, 1.0, 100.0, 1e-3])):
        case.check("lambda", lam=lam)
        case.check("lambda of the type", lam=lam.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_long_caches(dtype):
    # more than 64 entries of a table a wave, more than one workgroup a request
    Case([16384, 9001], 1, 16, 4, 1, 64, 64, dtype, 150).check("long")
    Case([16384], 20, 16, 2, 1, 32, 64, dtype, 160, _tree_masks(1, 20, 9)).check("long tree")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 20])
def test_requests_of_very_different_lengths(n, dtype):
    # more requests than a wave has lanes, some of them in several parts
    rng = random.Random(n)
    lengths = [rng.choice([0, 1, 3, 40, 333, 900]) for _ in range(130)]
    counts = [rng.choice([0, 1, n, n]) for _ in range(130)]
    Case(lengths, n, 16, 1, 1, 32, 64, dtype, 170, counts=counts).check("many requests")
    Case([12000] + [0] * 7, n, 32, 4, 2, 64, 64, dtype, 180, counts=[n] + [0, 1] * 3 + [n]).check("one long one")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 5, 40])
def test_long_parts_with_holes(n, dtype):
    # parts of more tiles than a wave reads of the table at once, and pages that are not there among them
    case = Case([5000, 6100, 4444, 10, 2000, 5999, 17, 3000], n, 16, 32, 8, 64, 64, dtype, 190, spare=0)
    for request, slot in ((0, 150), (0, 151), (1, 0), (1, 381), (2, 33), (4, 124), (5, 200), (7, 187)):
        case.table[request, slot] = -1
    case.check("holes")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [17, 33, 50, 65, 130, 200])
@pytest.mark.parametrize("d, dv", HEADS + [(24, 40), (40, 48), (40, 96), (72, 24), (72, 136), (24, 200)])
def test_rows_of_a_key_head(d, dv, n, dtype):
    # every way to share a tile among waves, for each size of heads and for heads below it
    Case([700, 33], n, 32, 1, 1, d, dv, dtype, 210).check("%d rows" % n)


@pytest.mark.parametrize("d, dv, n", [(128, 256, 9), (128, 256, 33), (64, 128, 17), (128, 128, 12)])
def test_long_parts_of_wide_heads(d, dv, n):
    for dtype in TYPES:
        Case([3001, 4100], n, 48, 4, 1, d, dv, dtype, 200, _tree_masks(2, n, n)).check("tree")


def test_offsets_past_32_bits():
    # pages beyond 2^32 bytes and elements: 2^33 bytes of keys
    pages, page, d = 2 ** 33 // (16 * 2 * 128 * 2 * 4), 16, 128
    k = torch.empty(pages, 4, page, 2, d, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(pages, 4, page, d, dtype=torch.bfloat16, device=DEV)
    assert k.numel() * 2 >= 2 ** 33 and k.numel() >= 2 ** 32
    case = Case([100, 40], 3, page, 4, 4, d, d, torch.bfloat16, 170)
    far = [pages - 1 - p for p in range(case.k.shape[0])]
    k[far], v[far] = case.k.to(DEV), case.v.to(DEV)
    table = torch.where(case.table >= 0, pages - 1 - case.table, -1).int().to(DEV)
    out = enc.diff_attention_pages(case.q.to(DEV), k, v, table, case.lengths.to(DEV), case.lam.to(DEV))
    case.check("far", out)
    # and the other calls there
    q, kn, vn = (t.to(DEV) for t in (case.q, _make((2, 3, 4, 2, d), torch.bfloat16, 171), _make((2, 3, 4, d), torch.bfloat16, 172)))
    enc.norm_rotate_append(q, kn, vn, k, v, table, case.lengths.to(DEV), norm=False)
    for b, length in enumerate((100, 40)):
        for i in range(3):
            p, at = int(table[b, (length + i) // page]), (length + i) % page
            assert torch.equal(k[p, :, at], kn[b, i]) and torch.equal(v[p, :, at], vn[b, i])
    enc.pages_compact(k, v, table, case.lengths.to(DEV), torch.tensor([[2], [1]], dtype=torch.int32, device=DEV))
    for b, (length, step) in enumerate(((100, 2), (40, 1))):
        p, at = int(table[b, length // page]), length % page
        assert torch.equal(k[p, :, at], kn[b, step]) and torch.equal(v[p, :, at], vn[b, step])
    enc.pages_copy(k, v, torch.tensor([[far[0], 0], [1, far[1]]], dtype=torch.int32, device=DEV))
    assert torch.equal(k[0], k[far[0]]) and torch.equal(v[far[1]].view(torch.int16), v[1].view(torch.int16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_strided_queries(offset, dtype):
    case = Case([50, 300], 6, 16, 4, 2, 64, 128, dtype, 180)
    wide = torch.zeros(2, 6, 4 * 2 * 64 + 5, dtype=dtype, device=DEV)
    wide[..., offset:offset + 512] = case.q.to(DEV).flatten(2)
    case.check("view", case.run(wide[..., offset:offset + 512].unflatten(-1, (4, 2, 64))))
    case.check("heads first", case.run(case.q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)))
    case.check("last dimension apart", case.run(case.q.to(DEV).transpose(3, 4).contiguous().transpose(3, 4)))
    case.q = case.q[:1, :1].expand(2, 6, 4, 2, 64)
    case.check("broadcast", case.run(case.q[:1, :1].contiguous().to(DEV).expand(2, 6, 4, 2, 64)))


@pytest.mark.parametrize("dtype", TYPES)
def test_pages_in_common(dtype):
    # two requests with the same pages, one of them shorter; a page twice in one table
    case = Case([100, 100, 60], 1, 16, 4, 2, 64, 128, dtype, 190)
    case.table[1] = case.table[0]
    case.lengths[1] = 77
    case.table[2, 1] = case.table[2, 0]
    case.check("common pages")


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_calls(dtype):
    for b, n, h, hk, slots, pages in ((0, 1, 2, 2, 3, 4), (2, 0, 2, 2, 3, 4), (2, 1, 0, 2, 3, 4), (2, 3, 2, 2, 0, 4), (2, 3, 2, 2, 3, 0)):
        q = torch.ones(b, n, h, 2, 64, dtype=dtype, device=DEV)
        out = enc.diff_attention_pages(q, torch.ones(pages, hk, 16, 2, 64, dtype=dtype, device=DEV), torch.ones(pages, hk, 16, 128, dtype=dtype, device=DEV),
                                       torch.full((b, slots), -1, dtype=torch.int32, device=DEV), torch.full((b,), 9, dtype=torch.int32, device=DEV), torch.ones(h, dtype=dtype, device=DEV))
        assert out.shape == (b, n, h, 128) and not out.any()


def test_as_the_attention_over_dense_keys():
    case = Case([0, 60, 500, 1111], 4, 64, 8, 2, 64, 128, torch.float32, 200)
    tokens = 1111 + 4
    k, v = (pref.dense(t, case.table, tokens).to(DEV) for t in (case.k, case.v))
    want = enc.diff_attention(case.q.to(DEV), k, v, case.lam.to(DEV), causal=True, lengths=(case.lengths + 4).to(DEV), starts=case.lengths.to(DEV))
    # both within 2^-24 times the depth of their sums of the same values: scores of 64 terms, softmaxes, 1115 values
    assert (case.run() - want).abs().max() <= 1e-5 * want.abs().max()


def test_same_bits_on_every_call():
    case = Case([5000, 300], 17, 16, 8, 2, 64, 128, torch.bfloat16, 210)
    first = case.run()
    for _ in range(3):
        assert torch.equal(case.run(), first)


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("d, dv", HEADS)
@pytest.mark.parametrize("n, h", [(4, 8), (5, 8), (9, 8), (19, 8), (40, 8), (70, 8)])
def test_the_first_maps_probabilities_at_any_number_of_rows(n, h, d, dv, dtype):
    # Without the second map a result errs by its own rounding, by what 32 bits cost (the same operands in fp32) and by what two parts of 8 or 11 bits leave of a probability: 2^-16 or 2^-22 of it,
    # of fp16 half the spacing of its smallest numbers.  One part alone would leave 2^-8 or 2^-11.
    case = Case([300, 37, 0], n, 16, h, 2, d, dv, dtype, seed=n)
    lam = torch.zeros(h)
    args = case.table, case.lengths, lam, None, None, case.masks
    want = pref.PagesAttention(case.q.float(), case.k.float(), case.v.float(), *args)
    sizes = pref.PagesAttention(case.q.float(), case.k.float(), case.v.abs().float(), *args).out
    bound = want.out_bound + ref.UNIT[dtype] * want.out.abs() + ref.UNIT[dtype] ** 2 * sizes + ref.TINY[dtype]
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25 * want.seen.sum(-1)[:, :, None, None] * case.v.abs().max().double()
    ref.assert_within(case.run(lam=lam.to(DEV)), want.out, bound, "one map")
